"""Routed experts by ragged groups, and products in 8-bit floating point with a scale for each block of 128, as cases to be timed
and compared: what a served model with many experts does between its router and the sum of what the experts answer.

* `quantise`: rows of activations as e4m3 values with a scale for every 128 neighbouring values of a row: scale = max(m, 2^-100) / 448 in
  32 bits, m the largest magnitude of the 128, q = v / scale rounded to e4m3, half to even.
* `product`: out[r, n] = sum over the blocks b of 128 k of scale_a[r, b] * scale_w[n / 128, b] * sum_(k in b) qa[r, k] qw[n, k] (+ bias), or
  with `glu` silu(gate) * up of the two stacked halves of the weight's rows.
* `group`: the (row, choice) pairs of a step in the order of their experts (pairs of one expert in their own order): where every expert's
  pairs begin, which pair lies where, and where each pair went. A choice of -1 is no expert (a row that fills a batch up).
* `grouped`: every pair's row times its expert's weight, out[p] = a[row of p] @ w[expert of p]^T, in bfloat16 or in 8 bits as above.
* `experts`: the whole feed-forward: pairs grouped, gate and up product with the gated unit, down product, and of every row's answers the
  sum with the router's weights (in 8 bits rows and units are quantised in between).
"""
import math

import torch

own = False

DEVICE = "cuda:0"


# ---- the cases ----------------------------------------------------------------------------------------------------

def _named(name, case):
    return dict(case, name=name) if name else case


def _quantise(name, rows, dim, dtype):
    return _named(name, dict(op="quantise", rows=rows, dim=dim, dtype=dtype))


def _product(name, rows, width, dim, *, glu=False, bias=False, dtype="bfloat16"):
    """`width`: the weight's rows (gate and up rows together with `glu`), `dim`: the sum's length."""
    return _named(name, dict(op="product", rows=rows, width=width, dim=dim, glu=glu, bias=bias, dtype=dtype))


def _group(name, rows, top, experts, unused=0.0):
    return _named(name, dict(op="group", rows=rows, top=top, experts=experts, unused=unused))


def _grouped(name, kind, rows, top, experts, width, dim, *, glu=False, dtype="bfloat16", unused=0.0):
    return _named(name, dict(op="grouped", kind=kind, rows=rows, top=top, experts=experts, width=width, dim=dim, glu=glu, dtype=dtype, unused=unused))


def _experts(name, kind, rows, top, experts, dim, hidden):
    return _named(name, dict(op="experts", kind=kind, rows=rows, top=top, experts=experts, dim=dim, hidden=hidden, unused=0.0))


def listed():
    return [
        # eight requests' attention results in front of the output product
        _quantise("quantise 8", 8, 4096, "bfloat16"),
        # a prompt's gated units in front of the down product
        _quantise("quantise 2048 wide", 2048, 12288, "bfloat16"),
        # one user's chat: the output product of a decode step
        _product("product 1", 1, 4096, 4096),
        # a busy server: the down product of 64 requests
        _product("product 64 down", 64, 4096, 12288),
        # odd sizes: rows, channels and sum length that no tile divides, with a bias and a float32 result
        _product("product 777 odd", 777, 1003, 2049, bias=True, dtype="float32"),
        # a prompt through gate and up: the largest product of a layer
        _product("product 2048 glu", 2048, 24576, 4096, glu=True),
        # eight requests' choices among 128 experts: only latency counts
        _group("group 8", 8, 8, 128),
        # a large batch of prompts, a part of it rows that fill the batch up
        _group("group 16384", 16384, 8, 256, unused=0.05),
        # a decode step's gate and up: eight requests, about fifty of 128 experts asked
        _grouped("grouped 8 bf16", "bfloat16", 8, 8, 128, 1536, 2048, glu=True),
        # a middle-sized prompt in 8 bits over odd sizes, some rows without experts
        _grouped("grouped 700 fp8 odd", "fp8", 700, 4, 60, 1407, 1930, dtype="float32", unused=0.1),
        # sixteen requests' whole feed-forward in 8 bits
        _experts("experts 16 fp8", "fp8", 16, 8, 128, 2048, 768),
        # a prompt's whole feed-forward
        _experts("experts 2048 bf16", "bfloat16", 2048, 8, 128, 2048, 768),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST_WEIGHTS = 400e6          # of all experts together
MOST_FLOPS = 100e9


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "product", "group", "grouped", "grouped", "grouped", "experts", "experts"])
    rows = _spread(rng, 1, 2048)
    if op == "quantise":
        return _quantise("", rows, _spread(rng, 64, 12288), rng.choice(["bfloat16", "float32"]))
    if op == "product":
        glu = rng.random() < 0.3
        width = 16 * _spread(rng, 4, 1536) if glu else _spread(rng, 64, 24576)
        dim = _spread(rng, 64, min(12288, 24576 * 4096 // width))
        return _product("", rows, width, dim, glu=glu, bias=not glu and rng.random() < 0.4,
                        dtype="bfloat16" if glu else rng.choice(["bfloat16", "float32"]))
    experts = _spread(rng, 4, 256)
    top = rng.randint(1, min(8, experts))
    if op == "group":
        return _group("", _spread(rng, 1, 16384), top, experts, unused=rng.choice([0.0, 0.1, 0.5]))
    kind = rng.choice(["bfloat16", "fp8"])
    experts = min(experts, 128)
    most = MOST_WEIGHTS / experts
    if op == "grouped":
        glu = rng.random() < 0.4
        width = 16 * _spread(rng, 8, 256) if glu else _spread(rng, 64, 4096)
        dim = _spread(rng, 64, int(min(4096, most / width)))
        if kind == "bfloat16":
            dim = max(64, dim // 8 * 8)
        rows = max(1, min(rows, int(MOST_FLOPS / (2 * top * width * dim))))
        return _grouped("", kind, rows, top, experts, width, dim, glu=glu, dtype="bfloat16" if glu else rng.choice(["bfloat16", "float32"]),
                        unused=rng.choice([0.0, 0.0, 0.2]))
    hidden, dim = 8 * _spread(rng, 8, 192), 8 * _spread(rng, 16, 512)
    dim = max(128, min(dim, int(most / 3 / hidden) // 8 * 8))
    rows = max(1, min(rows, int(MOST_FLOPS / (6 * top * hidden * dim))))
    return _experts("", kind, rows, top, experts, dim, hidden)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _random(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _activations(g, rows, dim):
    """Values as a part's result has them: rows of different sizes, and a few channels much larger than the others."""
    v = _random(g, rows, dim) * torch.exp(0.5 * _random(g, rows, 1))
    loud = torch.rand((dim,), generator=g, device=DEVICE) < 0.004
    return v * (1.0 + 19.0 * loud)


def _to_e4m3(x):
    """float64 `x` rounded to the nearest e4m3 value, half to even, as float64; magnitudes of 448 at most."""
    _, exponent = torch.frexp(x.abs())
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _blocks(v):
    """The last axis in blocks of 128, filled up with zeros."""
    dim = v.shape[-1]
    return torch.nn.functional.pad(v, (0, -dim % 128)).unflatten(-1, (-1, 128))


def _to_fp8(v):
    """e4m3 values [rows, dim] of float32 rows and their float32 scales [rows, blocks]."""
    b = _blocks(v)
    scale = (b.abs().amax(dim=-1).clamp(min=2.0 ** -100).double() / 448.0).float()          # (torch multiplies float32 by 1 / 448 instead)
    q = _to_e4m3(b.double() / scale.double()[..., None])
    return q.flatten(-2)[..., :v.shape[-1]].to(torch.float8_e4m3fn), scale


def _fp8_weight(g, *shape):
    """A weight as e4m3 values [..., rows, dim] and a scale for every 128 x 128 block of it."""
    *lead, rows, dim = shape
    scale = (0.5 + torch.rand((*lead, -(-rows // 128), -(-dim // 128)), generator=g, device=DEVICE)) * (dim ** -0.5 / 128.0)
    q = (_random(g, *shape) * 100.0).clamp_(-448.0, 448.0)
    return q.to(torch.float8_e4m3fn), scale


def _choices(g, case):
    """int32 [rows, top]: a row's experts, all different. Of many rows some experts are asked more than others (every one is asked still);
    a share of the rows has none."""
    rows, experts = case["rows"], case["experts"]
    score = -torch.log(-torch.log(torch.rand((rows, experts), generator=g, device=DEVICE).clamp_(min=1e-20, max=1.0 - 2.0 ** -24)))
    if rows * case["top"] >= 16 * experts:
        score = score + 0.5 * _random(g, experts)
    choice = score.topk(case["top"], dim=1).indices.to(torch.int32)
    if case["unused"]:
        choice[torch.rand((rows,), generator=g, device=DEVICE) < case["unused"]] = -1
    return choice


def _inputs(case, seed):
    """The case's inputs: what both forms and the 64-bit definition read."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, rows = case["op"], case["rows"]
    if op == "quantise":
        return dict(x=_activations(g, rows, case["dim"]).to(getattr(torch, case["dtype"])))
    if op == "product":
        s = dict(a=_to_fp8(_activations(g, rows, case["dim"])), weight=_fp8_weight(g, case["width"], case["dim"]), bias=None)
        if case["bias"]:
            s["bias"] = _random(g, case["width"]).to(torch.bfloat16)
        return s
    s = dict(choice=_choices(g, case))
    if op == "group":
        return s
    dim, experts = case["dim"], case["experts"]
    x = _activations(g, rows, dim).to(torch.bfloat16)

    def weight(width, dim):
        if case["kind"] == "fp8":
            return _fp8_weight(g, experts, width, dim)
        return (_random(g, experts, width, dim) * dim ** -0.5).to(torch.bfloat16)
    if op == "grouped":
        return dict(s, a=_to_fp8(x.float()) if case["kind"] == "fp8" else x, weight=weight(case["width"], dim))
    share = torch.softmax(_random(g, rows, case["top"]), dim=1)
    return dict(s, x=x, share=share, gate_up=weight(2 * case["hidden"], dim), down=weight(dim, case["hidden"]))


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    op, rows = case["op"], case["rows"]
    if op == "grouped":          # the plan of the step, made in front of its products
        s["plan"] = _plain_plan(s["choice"], case["experts"])
    if own:
        # what a serving program keeps: packed weights, the plan's room and the buffers of a step's results
        from jllm_serve_b200.csrc import ops

        def packed(weight, glu=False):
            return ops.pack_fp8(*weight, glu=glu) if isinstance(weight, tuple) else ops.pack_grouped(weight, glu=glu)
        if op == "quantise":
            s["rows8"] = ops.fp8_rows(rows, case["dim"], DEVICE)
            s["values"] = torch.empty((rows, case["dim"]), dtype=torch.bfloat16, device=DEVICE)
            return s
        if op == "product":
            s["packed"] = packed(s.pop("weight"), case["glu"])
            s["rows8"] = _rows8(ops, *s.pop("a"))
            s["out"] = torch.empty((rows, case["width"] // (2 if case["glu"] else 1)), dtype=getattr(torch, case["dtype"]), device=DEVICE)
            return s
        s["groups"] = ops.row_groups(rows, case["top"], case["experts"], DEVICE)
        if op == "grouped":
            ops.group_rows(s["choice"], s["groups"])
            s["packed"] = packed(s.pop("weight"), case["glu"])
            a = s.pop("a")
            s["rows"] = _rows8(ops, *a) if isinstance(a, tuple) else a
            width = case["width"] // (2 if case["glu"] else 1)
            s["out"] = torch.zeros((rows * case["top"], width), dtype=getattr(torch, case["dtype"]), device=DEVICE)
        if op == "experts":
            hidden, dim, pairs, fp8 = case["hidden"], case["dim"], rows * case["top"], case["kind"] == "fp8"
            s["packed"] = packed(s.pop("gate_up"), True), packed(s.pop("down"))
            if fp8:
                s["rows8"], s["units8"] = ops.fp8_rows(rows, dim, DEVICE), ops.fp8_rows(pairs, hidden, DEVICE)
            # (units that are rounded to 8 bits next are not rounded before)
            s["units"] = torch.empty((pairs, hidden), dtype=torch.float32 if fp8 else torch.bfloat16, device=DEVICE)
            s["answers"] = torch.empty((pairs, dim), device=DEVICE)          # (rounded once only, as their sum)
            s["out"] = torch.empty((rows, dim), dtype=torch.bfloat16, device=DEVICE)
    return s


def _rows8(ops, q, scale):
    rows8 = ops.fp8_rows(q.shape[0], q.shape[1], DEVICE)
    rows8.data.copy_(q)
    rows8.scale.copy_(scale)
    return rows8


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _run_own(s):
    from jllm_serve_b200.csrc import ops
    case = s["case"]
    op = case["op"]
    if op == "quantise":
        ops.quantize_fp8(s["x"], s["rows8"])
        return {"values": ops.fp8_values(s["rows8"], s["values"]), "scale": s["rows8"].scale}
    if op == "product":
        ops.gemm_fp8(s["rows8"], s["packed"], s["out"], s["bias"], swiglu="silu" if case["glu"] else False)
        return s["out"]
    groups = s["groups"]
    if op == "group":
        ops.group_rows(s["choice"], groups)
        return {"offsets": groups.offsets, "order": groups.order, "place": groups.place}
    if op == "grouped":
        ops.gemm_grouped(s["rows"], s["packed"], groups, s["out"], swiglu="silu" if case["glu"] else False)
        return s["out"]
    gate_up, down = s["packed"]
    rows, units = s["x"], s["units"]
    ops.group_rows(s["choice"], groups)
    if case["kind"] == "fp8":
        ops.quantize_fp8(rows, s["rows8"])
        rows = s["rows8"]
    ops.gemm_grouped(rows, gate_up, groups, units, swiglu="silu")
    if case["kind"] == "fp8":
        ops.quantize_fp8(units, s["units8"])
        units = s["units8"]
    ops.gemm_grouped(units, down, groups, s["answers"], by_pair=True)
    ops.combine_groups(s["answers"], groups, s["share"], s["out"])
    return s["out"]


# ---- the plain forms: elementary operations in 32 bits --------------------------------------------------------------

def _plain_group(choice, experts):
    flat = choice.flatten()
    pairs = flat.shape[0]
    key = torch.where(flat < 0, experts, flat.long())
    ordered, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(experts + 1, device=key.device)).to(torch.int32)
    place = torch.empty_like(order)
    place[order] = torch.arange(pairs, device=key.device)
    return {"offsets": offsets, "order": torch.where(ordered < experts, order, -1).to(torch.int32),
            "place": torch.where(flat < 0, -1, place).to(torch.int32).view(choice.shape)}


def _plain_plan(choice, experts):
    """(expert, its pairs) of every expert that is asked."""
    g = _plain_group(choice, experts)
    at = g["offsets"].tolist()
    return [(e, at[e], g["order"][at[e]:at[e + 1]].long()) for e in range(experts) if at[e] < at[e + 1]]


def _plain_fp8_rows(q, scale):
    return q.float() * scale.repeat_interleave(128, dim=1)[:, :q.shape[1]]


def _plain_fp8_weight(q, scale):
    return q.float() * scale.repeat_interleave(128, dim=0)[:q.shape[0]].repeat_interleave(128, dim=1)[:, :q.shape[1]]


def _plain_weight(weight, e):
    return _plain_fp8_weight(weight[0][e], weight[1][e]) if isinstance(weight, tuple) else weight[e].float()


def _plain_rows(a):
    return _plain_fp8_rows(*a) if isinstance(a, tuple) else a.float()


def _plain_glu(both):
    half = both.shape[1] // 2
    gate, up = both[:, :half], both[:, half:]
    return gate / (1.0 + torch.exp(-gate)) * up


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quantise":
        q, scale = _to_fp8(s["x"].float())
        return {"values": _plain_fp8_rows(q, scale).to(torch.bfloat16), "scale": scale}
    if op == "product":
        out = _plain_fp8_rows(*s["a"]) @ _plain_fp8_weight(*s["weight"]).t()
        if case["glu"]:
            out = _plain_glu(out)
        if s["bias"] is not None:
            out = out + s["bias"].float()
        return out.to(getattr(torch, case["dtype"]))
    if op == "group":
        return _plain_group(s["choice"], case["experts"])
    top = case["top"]
    if op == "grouped":
        a = _plain_rows(s["a"])
        out = torch.zeros((case["rows"] * top, case["width"] // (2 if case["glu"] else 1)), device=DEVICE)
        for e, at, pairs in s["plan"]:
            one = a[pairs // top] @ _plain_weight(s["weight"], e).t()
            out[at:at + len(pairs)] = _plain_glu(one) if case["glu"] else one
        return out.to(getattr(torch, case["dtype"]))
    fp8 = case["kind"] == "fp8"
    x = s["x"].float()
    if fp8:
        x = _plain_fp8_rows(*_to_fp8(x))
    out = torch.zeros((case["rows"], case["dim"]), device=DEVICE)
    for e, at, pairs in _plain_plan(s["choice"], case["experts"]):
        units = _plain_glu(x[pairs // top] @ _plain_weight(s["gate_up"], e).t())
        if fp8:
            units = _plain_fp8_rows(*_to_fp8(units))
        answers = units @ _plain_weight(s["down"], e).t()
        out[pairs // top] += answers * s["share"].flatten()[pairs][:, None]         # (a row asks an expert once)
    return out.to(torch.bfloat16)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

_BYTES = {"bfloat16": 2, "float32": 4}


def _asked(case):
    """Experts that are asked: of even choices the expected number."""
    return case["experts"] * (1.0 - (1.0 - case["top"] / case["experts"]) ** (case["rows"] * (1.0 - case["unused"])))


def _weight_bytes(kind, width, dim):
    return width * dim + 4 * -(-width // 128) * -(-dim // 128) if kind == "fp8" else 2 * width * dim


def _row_bytes(kind, dim):
    return dim + 4 * -(-dim // 128) if kind == "fp8" else 2 * dim


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "quantise":
        dim = case["dim"]
        return {"bytes": rows * (dim * _BYTES[case["dtype"]] + _row_bytes("fp8", dim)), "flops": rows * dim * 3}
    if op == "product":
        width, dim = case["width"], case["dim"]
        out = rows * (width // 2 if case["glu"] else width) * _BYTES[case["dtype"]]
        return {"bytes": rows * _row_bytes("fp8", dim) + _weight_bytes("fp8", width, dim) + out + (2 * width if case["bias"] else 0),
                "flops": 2 * rows * width * dim}
    pairs = rows * case["top"]
    if op == "group":
        return {"bytes": 12 * pairs + 4 * (case["experts"] + 1), "flops": 2 * pairs}
    kind, dim, used = case["kind"], case["dim"], rows * case["top"] * (1.0 - case["unused"])
    if op == "grouped":
        width = case["width"]
        out = used * (width // 2 if case["glu"] else width) * _BYTES[case["dtype"]]
        return {"bytes": rows * _row_bytes(kind, dim) + _asked(case) * _weight_bytes(kind, width, dim) + out + 4 * pairs,
                "flops": 2 * used * width * dim}
    hidden = case["hidden"]
    # what lies between the calls (units, answers) need not leave the device's caches
    return {"bytes": rows * dim * (2 + 2) + _asked(case) * (_weight_bytes(kind, 2 * hidden, dim) + _weight_bytes(kind, dim, hidden)) + 8 * pairs,
            "flops": 6 * used * hidden * dim}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_fp8(v):
    """The values that the rows of `v` (float64) stand for in 8 bits, and the scales (which are held in 32 bits)."""
    rows, dim = v.shape
    scales = []
    out = torch.empty_like(v)
    for lo in range(0, dim, 128):
        part = v[:, lo:lo + 128]
        scale = (part.abs().max(dim=1).values.clamp(min=2.0 ** -100) / 448.0).float().double()
        t = part / scale[:, None]
        grid = 2.0 ** (torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3.0)
        out[:, lo:lo + 128] = torch.round(t / grid) * grid * scale[:, None]
        scales.append(scale)
    return out, torch.stack(scales, dim=1)


def _exact_values(rows8):
    """Values of rows of e4m3 data with a scale for each 128 values of a row."""
    q, scale = rows8
    return q.to(torch.float64) * scale.double()[:, torch.arange(q.shape[1], device=q.device) // 128]


def _exact_weight(weight, e):
    if not isinstance(weight, tuple):
        return weight[e].double()
    q, scale = weight[0][e], weight[1][e].double()
    r, k = torch.arange(q.shape[0], device=q.device) // 128, torch.arange(q.shape[1], device=q.device) // 128
    return q.to(torch.float64) * scale[r][:, k]


def _exact_units(both):
    gate, up = both.chunk(2, dim=1)
    return gate * torch.sigmoid(gate) * up


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantise":
        values, scale = _exact_fp8(s["x"].double())
        return {"values": values, "scale": scale}
    if op == "product":
        out = _exact_values(s["a"]) @ _exact_weight(tuple(t[None] for t in s["weight"]), 0).T
        if s["bias"] is not None:
            out = out + s["bias"].double()
        return _exact_units(out) if case["glu"] else out
    if op == "group":
        return None
    choice, top = s["choice"].cpu(), case["top"]
    fp8 = case["kind"] == "fp8"
    if op == "grouped":
        a = _exact_values(s["a"]) if fp8 else s["a"].double()
        out = torch.zeros((case["rows"] * top, case["width"] // (2 if case["glu"] else 1)), dtype=torch.float64, device=DEVICE)
    else:
        a = s["x"].double()
        if fp8:
            a = _exact_fp8(a)[0]
        out = torch.zeros((case["rows"], case["dim"]), dtype=torch.float64, device=DEVICE)
    at = 0
    for e in range(case["experts"]):
        row, slot = (choice == e).nonzero(as_tuple=True)          # (in the order of the pairs)
        if not len(row):
            continue
        row, slot = row.to(DEVICE), slot.to(DEVICE)
        if op == "grouped":
            one = a[row] @ _exact_weight(s["weight"], e).T
            out[at:at + len(row)] = _exact_units(one) if case["glu"] else one
            at += len(row)
            continue
        units = _exact_units(a[row] @ _exact_weight(s["gate_up"], e).T)
        if fp8:
            units = _exact_fp8(units)[0]
        out.index_add_(0, row, units @ _exact_weight(s["down"], e).T * s["share"].double()[row, slot][:, None])
    return out
