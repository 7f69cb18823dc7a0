"""Linears in 8-bit integers, as cases to be timed and compared: what a layer of a served model does with int8 weights and
int8 activations, one scale a token and one a weight row (channel).

* `norm`: the residual's addition, the root-mean-square norm and its result as int8 rows: t = x + y, v = t / sqrt(mean(t^2) +
  eps) * gain, v in 8 bits.
* `quantise`: rows of a part's result in 8 bits (the attention's result, the gated units): nothing to norm in front of them.
* `product`: out = (qa @ qw^T) * scale_a[:, None] * scale_w[None, :] (+ bias), or with `glu` silu(gate) * up of two stacked
  halves of the weight's rows.
* `ffn`: the three as a layer's feed-forward runs them: norm, gate and up product, units in 8 bits, down product.

A row in 8 bits is q = round(v * 127 / max|v|), half to even, with the scale max|v| / 127.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6


# ---- the cases ----------------------------------------------------------------------------------------------------

def _norm(name, rows, dim, add):
    return _named(name, dict(op="norm", rows=rows, dim=dim, add=add))


def _quantise(name, rows, dim, dtype):
    return _named(name, dict(op="quantise", rows=rows, dim=dim, dtype=dtype))


def _product(name, rows, width, dim, *, glu=False, bias=False, dtype="bfloat16"):
    """`width`: the weight's rows (gate and up rows together with `glu`), `dim`: the sum's length."""
    return _named(name, dict(op="product", rows=rows, width=width, dim=dim, glu=glu, bias=bias, dtype=dtype))


def _ffn(name, rows, dim, hidden):
    return _named(name, dict(op="ffn", rows=rows, dim=dim, hidden=hidden))


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # one user's next token: the smallest norm, where only latency counts
        _norm("norm 1", 1, 4096, "bfloat16"),
        # a prompt of the benchmark's length behind a product that left bfloat16
        _norm("norm 2048", 2048, 4096, "bfloat16"),
        # a portion of 512 prompt tokens beside 32 riders at the larger layer size, nothing to add (a model's first norm)
        _norm("norm 544 alone", 544, 5120, "none"),
        # eight requests' attention results in front of the output product
        _quantise("quantise 8", 8, 4096, "bfloat16"),
        # a prompt's gated units in front of the down product
        _quantise("quantise 2048 wide", 2048, 12288, "bfloat16"),
        # one user's chat: the output product of a decode step
        _product("product 1", 1, 4096, 4096),
        # the headline batch of the benchmark: queries, keys and values of eight requests
        _product("product 8 qkv", 8, 6144, 4096),
        # a busy server: the down product of 64 requests
        _product("product 64 down", 64, 4096, 12288),
        # odd sizes: rows, channels and sum length that no tile divides, with a bias and a float32 result
        _product("product 777 odd", 777, 1003, 2049, bias=True, dtype="float32"),
        # a middle-sized prompt through gate and up
        _product("product 300 glu", 300, 24576, 4096, glu=True),
        # the benchmark's prompt through gate and up: the largest product of a layer
        _product("product 2048 glu", 2048, 24576, 4096, glu=True),
        # sixteen requests' whole feed-forward: four calls, one after the other
        _ffn("feed-forward 16", 16, 4096, 12288),
    ]


def _spread(rng, lo, hi):
    n = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    return n - 1 if n == 3072 else n         # (a size that no case has)


def draw(rng):
    op = rng.choice(["norm", "quantise", "product", "product", "product", "ffn"])
    rows = _spread(rng, 1, 2048)
    if op == "norm":
        return _norm("", rows, _spread(rng, 64, 12288), rng.choice(["bfloat16", "float32", "none"]))
    if op == "quantise":
        return _quantise("", rows, _spread(rng, 64, 24576), rng.choice(["bfloat16", "float32"]))
    if op == "ffn":
        return _ffn("", _spread(rng, 1, 1024), 16 * (2 * _spread(rng, 8, 160) - 1), 16 * (2 * _spread(rng, 16, 544) - 1))
    glu = rng.random() < 0.3
    width = 16 * (2 * _spread(rng, 4, 768) - 1) if glu else _spread(rng, 64, 24576)
    dim = _spread(rng, 64, min(17408, 24576 * 4096 // width))
    return _product("", rows, width, dim, glu=glu, bias=not glu and rng.random() < 0.4,
                    dtype="bfloat16" if glu else rng.choice(["bfloat16", "float32"]))


# ---- inputs -------------------------------------------------------------------------------------------------------

def _random(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _activations(g, rows, dim):
    """Values as a part's result has them: rows of different sizes, and a few channels much larger than the others."""
    v = _random(g, rows, dim) * torch.exp(0.5 * _random(g, rows, 1))
    loud = torch.rand((dim,), generator=g, device=DEVICE) < 0.004
    return v * (1.0 + 19.0 * loud)


def _to_int8(v):
    """int8 rows of `v` and their scales; a row's memory begins at a multiple of 16 bytes, as the engine's buffers have it."""
    m = v.abs().amax(dim=1)
    q = torch.zeros((v.shape[0], -(-v.shape[1] // 16) * 16), dtype=torch.int8, device=v.device)[:, :v.shape[1]]
    q.copy_(torch.round(v * (127.0 / m)[:, None]).clamp(-127, 127))
    return q, m / 127.0


def _weight(g, rows, dim):
    w = _random(g, rows, dim) * (dim ** -0.5)
    q, scale = _to_int8(w)
    return q.contiguous(), scale


def _inputs(case, seed):
    """The case's inputs: what both forms and the 64-bit definition read."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, rows, dim = case["op"], case["rows"], case["dim"]
    if op in ("norm", "ffn"):
        x = _activations(g, rows, dim)
        add = case.get("add", "bfloat16")
        y = None if add == "none" else (0.3 * _random(g, rows, dim)).to(getattr(torch, add))
        s = dict(x=x, y=y, gain=(1.0 + 0.2 * _random(g, dim)).to(torch.bfloat16))
        if op == "ffn":
            s["gate_up"], s["down"] = _weight(g, 2 * case["hidden"], dim), _weight(g, dim, case["hidden"])
        return s
    if op == "quantise":
        return dict(x=_activations(g, rows, dim).to(getattr(torch, case["dtype"])))
    s = dict(zip(("a", "a_scale"), _to_int8(_activations(g, rows, dim))), weight=_weight(g, case["width"], dim), bias=None)
    if case["bias"]:
        s["bias"] = _random(g, case["width"]).to(torch.bfloat16)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        # what a serving program keeps: packed weights, and the buffers of a step's results
        from jllm_serve_b200.csrc import ops
        op, rows, dim = case["op"], case["rows"], case["dim"]
        if op in ("norm", "ffn", "quantise"):
            s["rows8"] = ops.int8_rows(rows, dim, DEVICE)
            s["values"] = torch.empty((rows, dim), dtype=torch.bfloat16, device=DEVICE)
        if op in ("norm", "ffn"):
            s["total"] = torch.empty_like(s["x"])
        if op == "product":
            s["packed"] = ops.pack_int8(*s.pop("weight"), glu=case["glu"])
            s["out"] = torch.empty((rows, case["width"] // (2 if case["glu"] else 1)), dtype=getattr(torch, case["dtype"]), device=DEVICE)
            s["rows8"] = ops.Int8Rows(s["a"], s["a_scale"])
        if op == "ffn":
            s["packed"] = ops.pack_int8(*s.pop("gate_up"), glu=True), ops.pack_int8(*s.pop("down"))
            s["hidden"] = torch.empty((rows, case["hidden"]), device=DEVICE)      # (rounded once only, to 8 bits)
            s["hidden8"] = ops.int8_rows(rows, case["hidden"], DEVICE)
            s["out"] = torch.empty((rows, dim), dtype=torch.bfloat16, device=DEVICE)
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _run_own(s):
    from jllm_serve_b200.csrc import ops
    op = s["case"]["op"]
    if op == "norm":
        ops.add_rmsnorm_int8(s["x"], s["gain"], EPS, s["rows8"], y=s["y"], total=s["total"] if s["y"] is not None else None)
        return {"total": s["total"] if s["y"] is not None else s["x"], "values": ops.int8_values(s["rows8"], s["values"]), "scale": s["rows8"].scale}
    if op == "quantise":
        ops.quantize_int8(s["x"], s["rows8"])
        return {"values": ops.int8_values(s["rows8"], s["values"]), "scale": s["rows8"].scale}
    if op == "product":
        ops.gemm_int8(s["rows8"], s["packed"], s["out"], s["bias"], swiglu="silu" if s["case"]["glu"] else False)
        return s["out"]
    gate_up, down = s["packed"]
    ops.add_rmsnorm_int8(s["x"], s["gain"], EPS, s["rows8"], y=s["y"], total=s["total"])
    ops.gemm_int8(s["rows8"], gate_up, s["hidden"], swiglu="silu")
    ops.quantize_int8(s["hidden"], s["hidden8"])
    ops.gemm_int8(s["hidden8"], down, s["out"])
    return {"total": s["total"], "out": s["out"]}


# ---- the plain forms: elementary operations in 32 bits --------------------------------------------------------------

def _plain_int8(v):
    """(whole numbers as float32, scale) of the rows of `v`."""
    m = v.abs().amax(dim=1)
    return torch.round(v * (127.0 / m)[:, None]).clamp(-127, 127), m / 127.0


def _plain_norm(x, y, gain):
    t = x if y is None else x + y.float()
    v = t * torch.rsqrt((t * t).mean(dim=1, keepdim=True) + EPS) * gain.float()
    return t, v


def _plain_product(a, a_scale, w, w_scale):
    return (a.float() @ w.float().t()) * a_scale[:, None] * w_scale[None, :]


def _plain_glu(both):
    half = both.shape[1] // 2
    gate, up = both[:, :half], both[:, half:]
    return gate / (1.0 + torch.exp(-gate)) * up


def _run_plain(s):
    case = s["case"]
    if case["op"] == "norm":
        t, v = _plain_norm(s["x"], s["y"], s["gain"])
        q, scale = _plain_int8(v)
        return {"total": t, "values": (q * scale[:, None]).to(torch.bfloat16), "scale": scale}
    if case["op"] == "quantise":
        q, scale = _plain_int8(s["x"].float())
        return {"values": (q * scale[:, None]).to(torch.bfloat16), "scale": scale}
    if case["op"] == "product":
        out = _plain_product(s["a"], s["a_scale"], *s["weight"])
        if case["glu"]:
            out = _plain_glu(out)
        if s["bias"] is not None:
            out = out + s["bias"].float()
        return out.to(getattr(torch, case["dtype"]))
    t, v = _plain_norm(s["x"], s["y"], s["gain"])
    hidden = _plain_glu(_plain_product(*_plain_int8(v), *s["gate_up"]))
    return {"total": t, "out": _plain_product(*_plain_int8(hidden), *s["down"]).to(torch.bfloat16)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

_BYTES = {"bfloat16": 2, "float32": 4, "none": 0}


def work(case):
    op, rows, dim = case["op"], case["rows"], case["dim"]
    if op == "norm":
        add = _BYTES[case["add"]]
        # x (and y) in, the sum (where there is one) and the int8 values out; the gains and the scales
        return {"bytes": rows * dim * (4 + add + (4 if add else 0) + 1) + 2 * dim + 4 * rows, "flops": rows * dim * 6}
    if op == "quantise":
        return {"bytes": rows * dim * (_BYTES[case["dtype"]] + 1) + 4 * rows, "flops": rows * dim * 3}
    if op == "product":
        width = case["width"]
        out = rows * (width // 2 if case["glu"] else width) * _BYTES[case["dtype"]]
        return {"bytes": rows * dim + width * dim + 4 * rows + 4 * width + out + (2 * width if case["bias"] else 0),
                "flops": 2 * rows * width * dim}
    hidden = case["hidden"]
    # the rows between the four calls stay on the device's caches: the input, the two weights and the two results
    return {"bytes": rows * dim * (4 + 2 + 4 + 2) + 3 * hidden * dim + 4 * (3 * hidden + dim) + 2 * dim, "flops": 6 * rows * hidden * dim}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(v):
    """The values that the rows of `v` (float64) stand for in 8 bits, and the scales."""
    scale = v.abs().max(dim=1, keepdim=True).values / 127.0
    return torch.round(v / scale) * scale, scale[:, 0]


def exact(case, seed):
    s = {k: v for k, v in _inputs(case, seed).items()}
    if case["op"] in ("norm", "ffn"):
        t = s["x"].double()
        if s["y"] is not None:
            t = t + s["y"].double()
        v = t / torch.sqrt((t ** 2).sum(dim=1, keepdim=True) / t.shape[1] + EPS) * s["gain"].double()
        values, scale = _exact_rows(v)
        if case["op"] == "norm":
            return {"total": t, "values": values, "scale": scale}
        (gu, gu_scale), (down, down_scale) = s["gate_up"], s["down"]
        both = values @ (gu.double() * gu_scale.double()[:, None]).T
        gate, up = both.chunk(2, dim=1)
        units, _ = _exact_rows(gate * torch.sigmoid(gate) * up)
        return {"total": t, "out": units @ (down.double() * down_scale.double()[:, None]).T}
    if case["op"] == "quantise":
        values, scale = _exact_rows(s["x"].double())
        return {"values": values, "scale": scale}
    w, w_scale = s["weight"]
    out = (s["a"].double() * s["a_scale"].double()[:, None]) @ (w.double() * w_scale.double()[:, None]).T
    if s["bias"] is not None:
        out = out + s["bias"].double()
    if case["glu"]:
        gate, up = out.chunk(2, dim=1)
        out = gate * torch.sigmoid(gate) * up
    return out
