"""Every gated unit in every kernel of the grouped products and the products in 8-bit floating point (GPU), against 64 bits.

Tolerances, beside a sum's (`test_gpu_grouped.py`): an activation takes over its gate's error by its largest slope (silu, and z sigmoid(1.702 z): 1.1, GELU:
1.2), limits take it over as it is. The fast exponential of an argument t is off by 2 + 1.173 |t| units in the last place, GELU's argument itself by 2.5 units of
it (five roundings of half a unit, all terms of one sign); six units for quotient and products, two for u + 1. Where the exponential leaves float32 the value is
taken for zero: below 10^-35."""
import math

import pytest
import torch

from tests.test_gpu_grouped import (DEV, ULP, check, choices, fp8_weight, ops, plain_fp8, plain_groups, product_slack, rnd, rows_of, values_of,  # noqa: F401
                                    weight_values)

pytestmark = pytest.mark.gpu
LIMIT = 1.5
KINDS = ["silu", "gelu_tanh", "swish_clamped"]


def units(kind, both, slack):
    """(units, how far they may be off) of [rows, gate and up] and its slack, float64."""
    gate, up = both.chunk(2, dim=1)
    eg, eu = slack.chunk(2, dim=1)
    if kind == "silu":
        slope, t = 1.1, gate
        act = gate * torch.sigmoid(t)
    elif kind == "gelu_tanh":
        slope, t = 1.2, 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        act = gate * torch.sigmoid(t)
    else:
        gate, up = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT) + 1
        slope, t = 1.1, 1.702 * gate
        act = gate * torch.sigmoid(t)
        eu = eu + 2 * ULP * (1 + LIMIT)
    return act * up, slope * eg * (up.abs() + eu) + act.abs() * eu + (8 + 3.8 * t.abs()) * ULP * (act * up).abs() + 1e-35


def kernel_word(ops, kind):
    return ops.glu_descriptor(kind, LIMIT)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cut", [0, 16111, 16121, 32121, 64121, 16114, 16118, 32122, 128211, 128212, 128214])
@pytest.mark.parametrize("rows,hidden,k", [(5, 72, 1030), (33, 200, 640), (140, 136, 1500)])
def test_product(ops, kind, cut, rows, hidden, k):  # noqa: F811
    q, sq = plain_fp8(rnd(rows, k, seed=1) * torch.exp(rnd(rows, 1, seed=5)))
    wq, ws = fp8_weight(2 * hidden, k, 1)
    ws = ws * 2
    a, w = values_of(q, sq), weight_values(wq, ws)
    want, slack = units(kind, a @ w.T, product_slack(a, w, -(-k // 128)))
    packed, a8 = ops.pack_fp8(wq.to(DEV), ws.to(DEV), glu=True), rows_of(ops, q, sq)
    for dtype, pad in ((torch.float32, 0), (torch.float32, 3), (torch.bfloat16, 0), (torch.bfloat16, 1)):
        room = torch.full((rows, hidden + pad), 4.0, dtype=dtype, device=DEV)
        if cut % 10 > -(-k // 128):                    # (a cluster's blocks have a k block each at least)
            with pytest.raises(ops.KernelError, match="no clusters"):
                ops.gemm_fp8(a8, packed, room[:, pad:], swiglu=kernel_word(ops, kind), cut=cut)
            continue
        ops.gemm_fp8(a8, packed, room[:, pad:], swiglu=kernel_word(ops, kind), cut=cut)
        check(room[:, pad:], want, slack, dtype, f"{kind} {rows} x {hidden} x {k} cut {cut}")
        assert room[:, :pad].eq(4).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("values", ["bfloat16", "fp8"])
@pytest.mark.parametrize("cut", [0, 16111, 16121, 32121, 64121, 128211])
@pytest.mark.parametrize("by_pair", [False, True])
def test_groups(ops, kind, values, cut, by_pair):  # noqa: F811
    rows, top, groups, hidden, k = 120, 2, 5, 136, 520
    choice = choices(rows, top, groups)
    room = ops.row_groups(rows, top, groups, DEV)
    ops.group_rows(choice.to(DEV), room)
    offsets, order, _ = plain_groups(choice, groups)
    m = rows * top if by_pair else rows
    x = rnd(m, k, seed=2) * torch.exp(rnd(m, 1, seed=5))
    if values == "fp8":
        q, sq = plain_fp8(x)
        a, av = rows_of(ops, q, sq), values_of(q, sq)
        weights = [fp8_weight(2 * hidden, k, g) for g in range(groups)]
        packed = ops.pack_fp8(torch.stack([w[0] for w in weights]).to(DEV), torch.stack([2 * w[1] for w in weights]).to(DEV), glu=True)
        wv = [weight_values(w[0], 2 * w[1]) for w in weights]
    else:
        a, av = x.to(torch.bfloat16).to(DEV), x.to(torch.bfloat16).double()
        w = (torch.stack([rnd(2 * hidden, k, seed=g) for g in range(groups)]) * (2 / math.sqrt(k))).to(torch.bfloat16)
        packed, wv = ops.pack_grouped(w.to(DEV), glu=True), w.double()
    for dtype, pad in ((torch.float32, 3), (torch.bfloat16, 0)):
        out = torch.full((rows * top, hidden + pad), 5.0, dtype=dtype, device=DEV)
        ops.gemm_grouped(a, packed, room, out[:, pad:], swiglu=kernel_word(ops, kind), by_pair=by_pair, cut=cut)
        for g in range(groups):
            lo, hi = offsets[g], offsets[g + 1]
            if lo == hi:
                continue
            rows_g = av[lo:hi] if by_pair else av[[p // top for p in order[lo:hi]]]
            slack = product_slack(rows_g, wv[g], -(-k // 64)) if values == "fp8" else (k + 4) * ULP * (rows_g.abs() @ wv[g].abs().T)
            want, slack = units(kind, rows_g @ wv[g].T, slack)
            check(out[lo:hi, pad:], want, slack, dtype, f"{kind} {values} group {g} cut {cut}")
        assert out[offsets[-1]:].eq(5).all() and out[:, :pad].eq(5).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cut", [0, 16121, 32122, 64121, 128211, 128212])
def test_what_is_not_a_number_stays_so(ops, kind, cut):  # noqa: F811
    """Also through the limits of the clamped unit."""
    rows, hidden, k = 20, 72, 600
    x = rnd(rows, k)
    x[3, 130], x[17, 599] = math.nan, math.inf
    a8 = ops.fp8_rows(rows, k, DEV)
    ops.quantize_fp8(x.to(DEV), a8)
    wq, ws = fp8_weight(2 * hidden, k)
    out = torch.empty(rows, hidden, device=DEV)
    ops.gemm_fp8(a8, ops.pack_fp8(wq.to(DEV), ws.to(DEV), glu=True), out, swiglu=kernel_word(ops, kind), cut=cut)
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[[3, 17]] = True
    assert out[bad.to(DEV)].isnan().all() and out[(~bad).to(DEV)].isfinite().all()
