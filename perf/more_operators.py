"""Layers in 8-bit floating point, dense and by expert, and the way of rows to experts and back, as measurable cases.

`quantize`: rows of values, some of them several times and in another order, to E4M3 elements with a scale for each 128, and back.
`layer`: a dense layer on two such matrices, with bias and activation.
`experts`: the same for rows in groups of any sizes, each with weights of its own.
`route`: the experts of every row out of a router's logits, their shares, and the order of the rows by expert.
`combine`: every row's weighted sum of what its experts made of it.
`mixture`: all of them in a row, two layers an expert.

`listed()` names the cases to watch, `draw(rng)` gives others of the same ranges, `prepare` makes what a program has in hand
(packed weights, activations, logits, buffers that it keeps), `run` is one pass: the operators written out in elementary
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
BLOCK = 128


def listed():
    return [
        # four samples on their way to two experts each, in front of a layer: latency
        {"name": "quantize_8x8192_bf16", "kind": "quantize", "rows": 8, "cols": 8192, "source": 4, "pad": 0, "type": "bf16", "out": "bf16"},
        # a layer's weights, or the activations of a large batch: bandwidth
        {"name": "quantize_16384x8192_f32", "kind": "quantize", "rows": 16384, "cols": 8192, "source": 0, "pad": 0, "type": "f32", "out": "f32"},
        # the first layer of the large net for one sample: the weights are read once
        {"name": "layer_1x8192x16384_f32", "kind": "layer", "rows": 1, "in": 8192, "units": 16384, "act": "foo52", "out": "f32"},
        # a layer of the wide net on its batch: products
        {"name": "layer_16384x8192x8192_bf16", "kind": "layer", "rows": 16384, "in": 8192, "units": 8192, "act": "leaky", "out": "bf16"},
        # a served batch, a few rows an expert, some experts without any: the weights are read once
        {"name": "experts_64x32x4096x8192_f16", "kind": "experts", "rows": 64, "behind": 0, "experts": 32, "in": 4096, "units": 8192, "act": "relu", "out": "f16"},
        # a large batch in uneven groups, no size a multiple of a tile: products
        {"name": "experts_20011x12x4104x8001_bf16", "kind": "experts", "rows": 20011, "behind": 0, "experts": 12, "in": 4104, "units": 8001, "act": "leaky", "out": "bf16"},
        # one sample's experts: latency
        {"name": "route_1x64_f32", "kind": "route", "rows": 1, "experts": 64, "top": 2, "pad": 0, "type": "f32", "masked": 0.0, "normalise": True},
        # a large batch to eight of many experts, some of them closed to some rows
        {"name": "route_16384x256_bf16", "kind": "route", "rows": 16384, "experts": 256, "top": 8, "pad": 0, "type": "bf16", "masked": 0.1, "normalise": False},
        # a few rows of odd width: latency
        {"name": "combine_3x777_f32", "kind": "combine", "rows": 3, "top": 3, "width": 777, "missing": 0.2, "type": "f32", "out": "f32"},
        # a large batch: bandwidth
        {"name": "combine_16384x8192_bf16", "kind": "combine", "rows": 16384, "top": 2, "width": 8192, "missing": 0.0, "type": "bf16", "out": "bf16"},
        # one sample through two of sixteen experts
        {"name": "mixture_1x16x4096x8192x4096_bf16", "kind": "mixture", "rows": 1, "experts": 16, "top": 2, "in": 4096, "hidden": 8192, "units": 4096, "act": "foo52", "type": "bf16", "out": "bf16"},
        # a batch through two of eight experts
        {"name": "mixture_4096x8x4096x8192x4096_bf16", "kind": "mixture", "rows": 4096, "experts": 8, "top": 2, "in": 4096, "hidden": 8192, "units": 4096, "act": "leaky", "type": "bf16", "out": "bf16"},
    ]


def _size(rng, most, least=1):
    """A whole number, its logarithm spread evenly; one in three a multiple of 32."""
    v = int(round(math.exp(rng.uniform(math.log(least), math.log(most + 0.49)))))
    v = max(32, v // 32 * 32) if rng.random() < 0.33 and most >= 32 else v
    return max(least, min(most, v))


def draw(rng):
    kind = rng.choice(("quantize", "layer", "layer", "experts", "experts", "experts", "route", "combine", "mixture", "mixture"))
    if kind == "quantize":
        cols = _size(rng, 16384)
        rows = _size(rng, min(16384, (1 << 26) // cols))
        return {"kind": kind, "rows": rows, "cols": cols, "source": rng.choice((0, _size(rng, rows))), "pad": rng.choice((0, 0, 1, 8, 24)), "type": rng.choice(("f32", "f16", "bf16")),
                "out": rng.choice(("f32", "bf16"))}
    if kind == "layer":
        k, units = _size(rng, 16384), _size(rng, 16384)
        return {"kind": kind, "rows": _size(rng, max(1, min(16384, (1 << 26) // units, (1 << 39) // (k * units)))), "in": k, "units": units, "act": rng.choice(tuple(ACTS)),
                "out": rng.choice(("f32", "f16", "bf16"))}
    if kind == "experts":
        experts, k = _size(rng, 256), _size(rng, 8192, 16)
        units = _size(rng, max(1, min(8192, (1 << 29) // (experts * k))))
        rows = _size(rng, max(1, min(16384, (1 << 26) // units, (1 << 38) // (k * units))))
        return {"kind": kind, "rows": rows, "behind": rng.choice((0, 0, _size(rng, 200))), "experts": experts, "in": k, "units": units,
                "act": rng.choice(("relu", "leaky", "foo52", "none")), "out": rng.choice(("f32", "f16", "bf16"))}
    if kind == "route":
        experts = _size(rng, 512)
        return {"kind": kind, "rows": _size(rng, 16384), "experts": experts, "top": _size(rng, min(8, experts)), "pad": rng.choice((0, 0, 1, 8)), "type": rng.choice(("f32", "f16", "bf16")),
                "masked": rng.choice((0.0, round(rng.uniform(0.0, 0.9), 2))), "normalise": rng.choice((True, False))}
    if kind == "combine":
        width, top = _size(rng, 16384), _size(rng, 8)
        return {"kind": kind, "rows": _size(rng, max(1, min(16384, (1 << 27) // (width * top)))), "top": top, "width": width, "missing": rng.choice((0.0, round(rng.uniform(0.0, 0.9), 2))),
                "type": rng.choice(("f32", "f16", "bf16")), "out": rng.choice(("f32", "f16", "bf16"))}
    experts, k = _size(rng, 64, 2), _size(rng, 4096, 16)
    hidden = _size(rng, max(16, min(8192, (1 << 28) // (experts * k))), 16)
    units, top = _size(rng, max(1, min(4096, (1 << 28) // (experts * hidden)))), _size(rng, min(8, experts))
    return {"kind": kind, "rows": _size(rng, max(1, min(4096, (1 << 37) // (top * hidden * (k + units))))), "experts": experts, "top": top, "in": k, "hidden": hidden, "units": units,
            "act": rng.choice(("relu", "leaky", "foo52")), "type": rng.choice(("f32", "f16", "bf16")), "out": rng.choice(("f16", "bf16"))}


def _blocks(cols):
    return -(-cols // BLOCK)


def _with_rows(case):
    """How many of the experts have rows: one in eight has none where there are rows for all."""
    return max(1, min(case["rows"], case["experts"] - case["experts"] // 8))


def work(case):
    rows, kind = case["rows"], case["kind"]
    if kind == "quantize":
        cols = case["cols"]
        packed = rows * (cols + _blocks(cols))
        return {"bytes": (case["source"] or rows) * cols * BYTES[case["type"]] + 2 * packed + rows * cols * BYTES[case["out"]] + (4 * rows if case["source"] else 0), "flops": 2 * rows * cols}
    if kind == "layer" or kind == "experts":
        k, units, groups = case["in"], case["units"], _with_rows(case) if kind == "experts" else 1
        return {"bytes": (rows + groups * units) * (k + _blocks(k)) + 4 * groups * units + rows * units * BYTES[case["out"]], "flops": 2 * rows * k * units}
    if kind == "route":
        n = rows * case["experts"]
        return {"bytes": n * BYTES[case["type"]] + rows * case["top"] * 16 + 4 * case["experts"] + 4, "flops": 4 * n}
    if kind == "combine":
        n = rows * case["top"] * case["width"]
        return {"bytes": int(n * (1 - case["missing"])) * BYTES[case["type"]] + rows * case["width"] * BYTES[case["out"]] + 8 * rows * case["top"], "flops": 2 * n}
    k, hidden, units, top = case["in"], case["hidden"], case["units"], case["top"]
    groups = min(case["experts"], rows * top)
    weights = groups * (hidden * (k + _blocks(k)) + units * (hidden + _blocks(hidden)) + 4 * (hidden + units))
    return {"bytes": rows * (k * BYTES[case["type"]] + units * BYTES[case["out"]] + 4 * case["experts"] + 4 * top) + weights, "flops": 2 * rows * top * hidden * (k + units)}


# ---- the packed form --------------------------------------------------------------------------------------------------------

def _scales(x):
    """Scale byte of every block of 128 of x [rows][blocks * 128], and which blocks are finite."""
    v = x.view(x.shape[0], -1, BLOCK)
    fine = torch.isfinite(v).all(-1)
    a = torch.where(fine, v.abs().amax(-1), torch.ones_like(v[..., 0]))
    m, e = torch.frexp(a)                                       # a = m * 2^e, 0.5 <= m < 1: 448 is 0.875 * 2^9
    e = torch.where(a > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -127)).clamp(-127, 127)
    return e, fine


def _rounded(x, cols):
    """What the elements of x [rows][cols] stand for when they are held in 8 bits; in the type of x, exact but for the rounding."""
    rows = x.shape[0]
    v = torch.zeros(rows, _blocks(cols) * BLOCK, dtype=x.dtype, device=x.device)
    v[:, :cols] = x
    e, fine = _scales(v)
    unit = torch.exp2(e.to(torch.float64)).to(x.dtype).unsqueeze(-1)
    q = v.view(rows, -1, BLOCK)
    q = torch.where(fine.unsqueeze(-1), q, torch.zeros_like(q)) * torch.exp2(-e.to(torch.float64)).to(x.dtype).unsqueeze(-1)
    step = torch.exp2((torch.frexp(q)[1] - 1).clamp(min=-6).to(x.dtype) - 3)
    q = torch.round(q / step) * step * unit
    return torch.where(fine.unsqueeze(-1), q, torch.full_like(q, math.nan)).view(rows, -1)[:, :cols]


def _pitch(cols):
    return -(-cols // 16) * 16


def _room(rows, cols):
    """Codes [rows][pitch] and scales: of four blocks of a row side by side, the rows behind one another, then the next four blocks."""
    return {"codes": torch.zeros(rows, _pitch(cols), dtype=torch.uint8, device="cuda"),
            "scales": torch.zeros(-(-_blocks(cols) // 4), rows, 4, dtype=torch.uint8, device="cuda"), "rows": rows, "cols": cols}


def _fill(m, first, x):
    """x as rows first .. of m"""
    rows, cols = x.shape
    blocks = _blocks(cols)
    v = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols))
    e, _ = _scales(v)
    q = v.view(rows, blocks, BLOCK) * torch.exp2(-e.float()).unsqueeze(-1)
    m["codes"][first:first + rows, :cols] = q.to(torch.float8_e4m3fn).view(torch.uint8).view(rows, -1)[:, :cols]
    byte = torch.zeros(rows, -(-blocks // 4) * 4, dtype=torch.uint8, device=x.device)
    byte[:, :blocks] = (e + 127).to(torch.uint8)
    m["scales"][:, first:first + rows] = byte.view(rows, -1, 4).transpose(0, 1)


def _values(m, first=0, rows=None):
    """Rows of a packed matrix as what they stand for, in 32 bits."""
    rows = m["rows"] if rows is None else rows
    cols, blocks = m["cols"], _blocks(m["cols"])
    table = torch.arange(256, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).float()
    v = torch.zeros(rows, blocks * BLOCK, device="cuda")
    v[:, :cols] = table[m["codes"][first:first + rows, :cols].long()]
    e = m["scales"][:, first:first + rows].transpose(0, 1).reshape(rows, -1)[:, :blocks]
    s = torch.exp2(e.double() - 127).float()
    s = torch.where(e == 255, torch.full_like(s, math.nan), s)
    return (v.view(rows, blocks, BLOCK) * s.unsqueeze(-1)).view(rows, -1)[:, :cols]


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _activations(rows, cols, g):
    """Values whose columns differ in size, as a layer's outputs do."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    return x * torch.exp2(torch.randn(1, cols, device="cuda", generator=g))


def _weights(groups, units, k, g):
    m = _room(groups * units, k)
    for e in range(groups):
        _fill(m, e * units, torch.randn(units, k, device="cuda", generator=g) / math.sqrt(k))
    return m, torch.randn(groups * units, device="cuda", generator=g) * 0.1


def _packed(rows, cols, g):
    m = _room(rows, cols)
    for i in range(0, rows, 8192):
        _fill(m, i, _activations(min(8192, rows - i), cols, g))
    return m


def _starts(case, seed):
    """Where the groups begin: sizes that differ by some factors, one expert in eight without rows."""
    rng = np.random.default_rng(seed)
    some = rng.permutation(case["experts"])[:_with_rows(case)]
    share = np.exp(rng.normal(0, 0.7, len(some)))
    counts = np.zeros(case["experts"], np.int64)
    counts[some] = 1 + rng.multinomial(case["rows"] - len(some), share / share.sum())
    return torch.from_numpy(np.concatenate(([0], np.cumsum(counts)))).to(torch.int32).cuda()


def _logits(rows, experts, pad, g):
    return torch.randn(rows, experts + pad, device="cuda", generator=g) * 1.5 + 0.5 * torch.randn(1, experts + pad, device="cuda", generator=g)


def _route_room(rows, experts, top):
    def ints(*shape):
        return torch.empty(*shape, dtype=torch.int32, device="cuda")
    return {"chosen": ints(rows, top), "gates": torch.empty(rows, top, device="cuda"), "starts": ints(experts + 1), "order": ints(rows * top), "places": ints(rows, top)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, kind = case["rows"], case["kind"]
    s = {"case": case}
    if kind == "quantize":
        cols, source = case["cols"], case["source"] or rows
        s["x"] = _activations(source, cols + case["pad"], g).to(TYPES[case["type"]])[:, :cols]
        s["index"] = torch.randint(0, source, (rows,), device="cuda", generator=g).to(torch.int32) if case["source"] else None
        s["packed"] = _room(rows, cols)
        s["y"] = torch.empty(rows, cols, dtype=TYPES[case["out"]], device="cuda")
    elif kind == "layer":
        s["w"], s["bias"] = _weights(1, case["units"], case["in"], g)
        s["x"] = _packed(rows, case["in"], g)
        s["y"] = torch.empty(rows, case["units"], dtype=TYPES[case["out"]], device="cuda")
    elif kind == "experts":
        s["w"], s["bias"] = _weights(case["experts"], case["units"], case["in"], g)
        s["x"] = _packed(rows + case["behind"], case["in"], g)
        s["starts"] = _starts(case, seed)
        s["y"] = torch.zeros(rows + case["behind"], case["units"], dtype=TYPES[case["out"]], device="cuda")       # rows behind the last group stay as they are
    elif kind == "route":
        full = _logits(rows, case["experts"], case["pad"], g)
        if case["masked"]:
            hidden = torch.rand(full.shape, device="cuda", generator=g) < case["masked"]
            if rows >= 8:
                hidden[rows // 3] = True                        # a row that no expert is open to
            full = full.masked_fill(hidden, float("-inf"))
        s["x"] = full.to(TYPES[case["type"]])[:, :case["experts"]]
        s["route"] = _route_room(rows, case["experts"], case["top"])
    elif kind == "combine":
        top, width = case["top"], case["width"]
        s["x"] = _activations(rows * top, width, g).to(TYPES[case["type"]])
        places = torch.randperm(rows * top, device="cuda", generator=g).to(torch.int32)
        s["places"] = torch.where(torch.rand(rows * top, device="cuda", generator=g) < case["missing"], torch.full_like(places, -1), places).view(rows, top)
        s["gates"] = torch.rand(rows, top, device="cuda", generator=g)
        s["y"] = torch.empty(rows, width, dtype=TYPES[case["out"]], device="cuda")
    else:
        experts, top = case["experts"], case["top"]
        s["w1"], s["bias1"] = _weights(experts, case["hidden"], case["in"], g)
        s["w2"], s["bias2"] = _weights(experts, case["units"], case["hidden"], g)
        s["x"] = _activations(rows, case["in"], g).to(TYPES[case["type"]])
        s["logits"] = _logits(rows, experts, 0, g)
        s["route"] = _route_room(rows, experts, top)
        s["x8"], s["h8"] = _room(rows * top, case["in"]), _room(rows * top, case["hidden"])
        s["z"] = torch.empty(rows * top, case["units"], dtype=TYPES[case["out"]], device="cuda")
        s["y"] = torch.empty(rows, case["units"], dtype=TYPES[case["out"]], device="cuda")
    if kind in ("layer", "experts", "mixture"):
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
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


def _by_expert(x, w, bias, units, act, starts, y):
    """y's rows of every group that has some, in the type of x."""
    at = starts.tolist()
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        if hi > lo:
            weights = _values(w, e * units, units).to(x.dtype)
            y[lo:hi] = _dense(x[lo:hi], weights, bias[e * units:(e + 1) * units].to(x.dtype), act).to(y.dtype)
    return y


def _route(x, top, normalise):
    rows, experts = x.shape
    l = x.float()
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l)
    most = l.amax(1, keepdim=True)
    w = torch.exp(l - torch.where(most > -math.inf, most, torch.zeros_like(most)))
    order = torch.sort(l, dim=1, descending=True, stable=True)[1][:, :top]
    open_ = torch.gather(l, 1, order) > -math.inf
    mine = torch.where(open_, torch.gather(w, 1, order), torch.zeros_like(l[:, :top]))
    total = (mine if normalise else w).sum(1, keepdim=True)
    gates = mine / torch.where(total > 0, total, torch.ones_like(total))
    chosen = torch.where(open_, order, torch.full_like(order, -1))
    flat = torch.where(open_, order, torch.full_like(order, experts)).view(-1)                # the closed ones last
    by_expert = torch.sort(flat, stable=True)[1]
    place = torch.empty_like(by_expert)
    place[by_expert] = torch.arange(rows * top, device=x.device)
    starts = torch.searchsorted(flat[by_expert], torch.arange(experts + 1, device=x.device))
    order = torch.where(torch.arange(rows * top, device=x.device) < starts[-1], by_expert // top, torch.full_like(by_expert, -1))
    places = torch.where(open_, place.view(rows, top), torch.full_like(chosen, -1))
    return {"chosen": chosen.to(torch.int32), "gates": gates, "starts": starts.to(torch.int32), "order": order.to(torch.int32), "places": places.to(torch.int32)}


def _combine(y, places, gates):
    out = torch.zeros(places.shape[0], y.shape[1], device=y.device)
    for j in range(places.shape[1]):
        p = places[:, j].long()
        out += torch.where((p >= 0).unsqueeze(1), gates[:, j:j + 1] * y[p.clamp(min=0)].float(), torch.zeros_like(out))
    return out


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        x = s["x"].float() if s["index"] is None else s["x"][s["index"].long()].float()
        return _rounded(x, case["cols"]).to(TYPES[case["out"]])
    if kind == "layer":
        return _dense(_values(s["x"]), _values(s["w"]), s["bias"], case["act"]).to(TYPES[case["out"]])
    if kind == "experts":
        return _by_expert(_values(s["x"]), s["w"], s["bias"], case["units"], case["act"], s["starts"], torch.zeros_like(s["y"]))
    if kind == "route":
        return _route(s["x"], case["top"], case["normalise"])
    if kind == "combine":
        return _combine(s["x"], s["places"], s["gates"]).to(TYPES[case["out"]])
    r = _route(s["logits"], case["top"], True)
    x = _rounded(s["x"].float(), case["in"])[r["order"].clamp(min=0).long()]
    # the hidden layer in 64 bits: its values are rounded to few of them, and some lie next to a border
    h = torch.zeros(x.shape[0], case["hidden"], dtype=torch.float64, device="cuda")
    h = _rounded(_by_expert(x.double(), s["w1"], s["bias1"], case["hidden"], case["act"], r["starts"], h), case["hidden"])
    z = _by_expert(h.float(), s["w2"], s["bias2"], case["units"], "none", r["starts"], torch.zeros(x.shape[0], case["units"], device="cuda"))
    # the experts' rows are kept in the output's type
    return {"y": _combine(z.to(TYPES[case["out"]]), r["places"], r["gates"]).to(TYPES[case["out"]]), "chosen": r["chosen"]}


def _handles(s):
    """The library and what its calls take, made once as a program would."""
    import ctypes
    import spingalett_b200 as spg

    lib = spg.lib()

    def matrix(m):
        return ctypes.byref(spg.abi.Fp8(m["codes"].data_ptr(), m["scales"].data_ptr(), m["rows"], m["cols"], m["codes"].shape[1]))

    def at(t):
        return None if t is None else t.data_ptr()

    case = s["case"]
    kind, rows = case["kind"], case["rows"]
    calls = []
    if kind == "quantize":
        packed = matrix(s["packed"])
        calls += [(lib.spgk_fp8_quantize, (at(s["x"]), CODES[case["type"]], s["x"].stride(0), s["x"].shape[0], at(s["index"]), packed)),
                  (lib.spgk_fp8_dequantize, (packed, at(s["y"]), CODES[case["out"]], case["cols"]))]
    elif kind == "layer":
        calls += [(lib.spgk_layer_fp8, (matrix(s["w"]), at(s["bias"]), ACTS[case["act"]], matrix(s["x"]), at(s["y"]), CODES[case["out"]], case["units"], None, at(s["status"])))]
    elif kind == "experts":
        calls += [(lib.spgk_experts_fp8, (matrix(s["w"]), case["experts"], at(s["bias"]), ACTS[case["act"]], matrix(s["x"]), at(s["starts"]), at(s["y"]), CODES[case["out"]], case["units"], None,
                                          at(s["status"])))]
    elif kind == "route":
        r = s["route"]
        calls += [(lib.spgk_route_rows, (at(s["x"]), CODES[case["type"]], s["x"].stride(0), rows, case["experts"], case["top"], int(case["normalise"]), at(r["chosen"]), at(r["gates"]),
                                         at(r["starts"]), at(r["order"]), at(r["places"])))]
    elif kind == "combine":
        calls += [(lib.spgk_combine_rows, (at(s["x"]), CODES[case["type"]], case["width"], rows * case["top"], at(s["places"]), at(s["gates"]), rows, case["top"], case["width"], at(s["y"]),
                                           CODES[case["out"]], case["width"]))]
    else:
        r, x8, h8, experts, top, out = s["route"], matrix(s["x8"]), matrix(s["h8"]), case["experts"], case["top"], CODES[case["out"]]
        calls += [(lib.spgk_route_rows, (at(s["logits"]), CODES["f32"], experts, rows, experts, top, 1, at(r["chosen"]), at(r["gates"]), at(r["starts"]), at(r["order"]), at(r["places"]))),
                  (lib.spgk_fp8_quantize, (at(s["x"]), CODES[case["type"]], case["in"], rows, at(r["order"]), x8)),
                  (lib.spgk_experts_fp8, (matrix(s["w1"]), experts, at(s["bias1"]), ACTS[case["act"]], x8, at(r["starts"]), None, 0, 0, h8, at(s["status"]))),
                  (lib.spgk_experts_fp8, (matrix(s["w2"]), experts, at(s["bias2"]), ACTS["none"], h8, at(r["starts"]), at(s["z"]), out, case["units"], None, at(s["status"]))),
                  (lib.spgk_combine_rows, (at(s["z"]), out, case["units"], rows * top, at(r["places"]), at(r["gates"]), rows, top, case["units"], at(s["y"]), out, case["units"]))]
    return lib, calls


def _library(s):
    if "calls" not in s:
        s["calls"] = _handles(s)
    lib, calls = s["calls"]
    stream = torch.cuda.current_stream().cuda_stream
    for call, args in calls:
        if call(*args, stream) != 0:
            raise RuntimeError(lib.spgk_error_string().decode())
    if s["case"]["kind"] == "route":
        return dict(s["route"])
    if s["case"]["kind"] == "mixture":
        return {"y": s["y"], "chosen": s["route"]["chosen"]}
    return s["y"]


def run(s):
    return _library(s) if own else _plain(s)


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------------

def _exact_values(m, first=0, rows=None):
    """Rows of a packed matrix read element by element from the description of its layout."""
    rows, cols = m["rows"] if rows is None else rows, m["cols"]
    c = m["codes"][first:first + rows, :cols].long()
    e, f = (c >> 3) & 15, (c & 7).double()
    size = torch.where(e == 0, f * 2.0 ** -9, torch.exp2(e.double() - 7) * (1 + f / 8))
    size = torch.where(c & 127 == 127, torch.full_like(size, math.nan), size)
    b = torch.arange(cols, device="cuda") // BLOCK
    r = torch.arange(first, first + rows, device="cuda").unsqueeze(1)
    byte = m["scales"].view(-1)[((b // 4).unsqueeze(0) * m["rows"] + r) * 4 + (b % 4).unsqueeze(0)].double()
    return torch.where(c & 128 != 0, -size, size) * torch.where(byte == 255, torch.full_like(byte, math.nan), torch.exp2(byte - 127))


def _exact_rounding(x):
    """Every value of x rounded to its block's grid, the nearest of the numbers that a code has, of two equally near ones that with the even code."""
    rows, cols = x.shape
    codes = torch.arange(127, device=x.device)
    sizes = torch.where(codes < 8, codes * 2.0 ** -9, (8 + codes % 8) * torch.exp2((codes // 8).double() - 10))
    v = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).view(-1, BLOCK)
    out = torch.empty_like(v)
    for i in range(0, v.shape[0], 1 << 18):
        p = v[i:i + (1 << 18)]
        a = p.abs().amax(1, keepdim=True)
        bad = ~torch.isfinite(p).all(1, keepdim=True)
        e = torch.ceil(torch.log2((a / 448).clamp(min=2.0 ** -127))).clamp(-127, 127)
        e = torch.where(a > 448 * torch.exp2(e), e + 1, e)
        e = torch.where((e > -127) & (a <= 448 * torch.exp2(e - 1)), e - 1, e)
        q = torch.where(bad, torch.zeros_like(p), p.abs() / torch.exp2(e))
        hi = torch.searchsorted(sizes, q.contiguous()).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        up, down = sizes[hi] - q, q - sizes[lo]
        at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        got = torch.copysign(sizes[at], p) * torch.exp2(e)
        out[i:i + (1 << 18)] = torch.where(bad, torch.full_like(got, math.nan), got)
    return out.view(rows, -1)[:, :cols]


def _exact_act(v, act):
    f = {"relu": lambda: v.clamp(min=0), "leaky": lambda: torch.maximum(v, 0.01 * v), "tanh": lambda: torch.tanh(v), "sigmoid": lambda: torch.sigmoid(v), "none": lambda: v,
         "foo52": lambda: v.clamp(0, 1) + 0.01 * (v - v.clamp(0, 1))}
    return f[act]()


def _exact_dense(x, w, bias, act):
    return _exact_act(torch.addmm(bias.double(), x, w.T), act)


def _exact_groups(x, w, bias, units, act, starts):
    out = torch.zeros(x.shape[0], units, dtype=torch.float64, device="cuda")
    for e in range(len(starts) - 1):
        if starts[e + 1] > starts[e]:
            rows = slice(starts[e], starts[e + 1])
            out[rows] = _exact_dense(x[rows], _exact_values(w, e * units, units), bias[e * units:(e + 1) * units], act)
    return out


def _exact_route(x, top, normalise):
    """Row by row: its experts by sorting; then one expert after the other, its rows as they come."""
    l = x.double().cpu().numpy()
    l = np.where(np.isnan(l), -np.inf, l)
    rows, experts = l.shape
    index = np.argsort(-l, axis=1, kind="stable")[:, :top]
    mine = np.take_along_axis(l, index, 1)
    chosen = np.where(mine > -np.inf, index, -1)
    most = np.where(np.isfinite(l.max(1, keepdims=True)), l.max(1, keepdims=True), 0.0)
    part = np.where(chosen >= 0, np.exp(mine - most), 0.0)
    whole = part.sum(1, keepdims=True) if normalise else np.exp(l - most).sum(1, keepdims=True)
    gates = part / np.where(whole > 0, whole, 1.0)
    order, places, starts = np.full(rows * top, -1), np.full((rows, top), -1), [0]
    for e in range(experts):
        n, j = np.nonzero(chosen == e)
        at = starts[-1] + np.arange(len(n))
        order[at], places[n, j] = n, at
        starts.append(starts[-1] + len(n))

    def ints(v):
        return torch.from_numpy(np.asarray(v, np.int32))
    return {"chosen": ints(chosen), "gates": torch.from_numpy(gates), "starts": ints(starts), "order": ints(order), "places": ints(places)}


def _exact_combine(y, places, gates):
    out = torch.zeros(places.shape[0], y.shape[1], dtype=torch.float64, device="cuda")
    for j in range(places.shape[1]):
        some = torch.nonzero(places[:, j] >= 0).squeeze(1)
        out.index_add_(0, some, y[places[some, j].long()].double() * gates[some, j].double().unsqueeze(1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _exact_rounding(s["x"] if s["index"] is None else s["x"].index_select(0, s["index"]))
    if kind == "layer":
        return _exact_dense(_exact_values(s["x"]), _exact_values(s["w"]), s["bias"], case["act"])
    if kind == "experts":
        return _exact_groups(_exact_values(s["x"]), s["w"], s["bias"], case["units"], case["act"], s["starts"].tolist())
    if kind == "route":
        return _exact_route(s["x"], case["top"], case["normalise"])
    if kind == "combine":
        return _exact_combine(s["x"], s["places"], s["gates"])
    r = _exact_route(s["logits"], case["top"], True)
    starts, order = r["starts"].tolist(), r["order"].cuda()
    h = _exact_groups(_exact_rounding(s["x"])[order.clamp(min=0).long()], s["w1"], s["bias1"], case["hidden"], case["act"], starts)
    z = _exact_groups(_exact_rounding(h), s["w2"], s["bias2"], case["units"], "none", starts)
    return {"y": _exact_combine(z, r["places"].cuda(), r["gates"].cuda()), "chosen": r["chosen"]}
