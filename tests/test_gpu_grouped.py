"""Products in 8-bit floating point and products of ragged groups of rows (GPU): every operator alone against plain forms in 64 bits, and
together as a layer's experts run them.

Tolerances. A rounding to a type is off by eps / 2 of the value. A product's float32 sum of n terms is off by at most n 2^-23 of the sum of their
magnitudes (every addition of the tensor cores and of the epilogue keeps 24 bits, cut off or rounded), scales by three roundings more. A gated unit
takes over its inputs' errors (|silu'| <= 1.1), and the fast exponential's: 2 + 1.173 |gate| units in the last place, and six units for the rest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ULP = 2.0 ** -23


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    yield o
    o.check_kernel_errors()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed + 7 * sum(shape)))


# ---- plain forms in 64 bits, on the CPU ----

def plain_e4m3(x):
    """float64 -> the nearest e4m3 value, half to even."""
    _, exponent = torch.frexp(x.abs())
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def plain_fp8(v):
    """(q float64 [rows, cols], scale float32 [rows, blocks]) of float32 rows."""
    rows, cols = v.shape
    blocks = torch.nn.functional.pad(v.double(), (0, -cols % 128)).view(rows, -1, 128)
    bad = ~torch.isfinite(blocks).all(dim=2)
    m = blocks.abs().amax(dim=2).clamp(min=2.0 ** -100)
    scale = (m / 448).float()
    q = plain_e4m3(torch.where(bad[..., None], torch.zeros_like(blocks), blocks) / torch.where(bad, torch.ones_like(m), scale.double())[..., None])
    return q.reshape(rows, -1)[:, :cols], torch.where(bad, torch.full_like(scale, math.nan), scale)


def values_of(q, scale):
    return q.double() * scale.double().repeat_interleave(128, dim=1)[:, :q.shape[1]]


def weight_values(q, scale):
    return q.double() * scale.double().repeat_interleave(128, dim=0)[:q.shape[0]].repeat_interleave(128, dim=1)[:, :q.shape[1]]


def fp8_weight(rows, cols, seed=0):
    q = (rnd(rows, cols, seed=seed) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = (0.25 + torch.rand((-(-rows // 128), -(-cols // 128)), generator=gen(seed + 3))) / (100 * math.sqrt(cols))
    return q, scale


def rows_of(ops, q, scale, dev=DEV):
    rows8 = ops.fp8_rows(q.shape[0], q.shape[1], dev)
    rows8.data.copy_(q.to(torch.float8_e4m3fn))
    rows8.scale.copy_(scale)
    return rows8


def check(got, want, slack, dtype, what=""):
    """|got - want| <= slack + a rounding to dtype"""
    bound = slack + (want.abs() + slack) * torch.finfo(dtype).eps / 2
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(off).all(), what
    worst = (off - bound).max()
    assert worst <= 0, f"{what}: {off.flatten()[(off - bound).argmax()]:.3e} off where {bound.flatten()[(off - bound).argmax()]:.3e} is allowed"


def product_slack(a, w, blocks):
    """of the product of a [rows, k] and w [n, k] (float64 values)"""
    return (128 + blocks + 4) * ULP * (a.abs() @ w.abs().T)


def units_and_slack(both, slack):
    gate, up = both.chunk(2, dim=1)
    eg, eu = slack.chunk(2, dim=1)
    silu = gate * torch.sigmoid(gate)
    return silu * up, 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + (8 + 1.2 * gate.abs()) * ULP * (silu * up).abs()


# ---- rows in 8 bits ----

@pytest.mark.parametrize("cols", [1, 7, 16, 127, 128, 129, 200, 512, 1000, 1930, 4096, 12288])
@pytest.mark.parametrize("rows", [1, 5, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantise_gives_the_plain_values(ops, rows, cols, dtype):
    x = (rnd(rows, cols) * torch.exp(rnd(rows, 1, seed=3))).to(dtype)
    q, scale = plain_fp8(x.float())
    out = ops.fp8_rows(rows, cols, DEV)
    ops.quantize_fp8(x.to(DEV), out)
    assert torch.equal(out.data.cpu().double(), q) and torch.equal(out.scale.cpu(), scale)
    for kind in (torch.float32, torch.bfloat16):
        got = ops.fp8_values(out, torch.empty((rows, cols), dtype=kind, device=DEV))
        assert torch.equal(got.cpu(), values_of(q, scale).float().to(kind))


def test_quantise_ties_and_their_neighbours(ops):
    """Quotients at every tie between two e4m3 values, and next to one: rounded once, whatever the scale's last bits are."""
    grid = torch.tensor(sorted({float(torch.tensor(i, dtype=torch.uint8).view(torch.float8_e4m3fn)) for i in range(127)}), dtype=torch.float64)
    ties = (grid[1:] + grid[:-1]) / 2
    rows = []
    for m in (448.0, 1.0, 3.0, 0.7, 1e-20, 1e20, 448.0 * 2.0 ** -100):
        scale = float(torch.tensor(m, dtype=torch.float64).float() / 1) / 448
        scale = float((torch.tensor(m).double() / 448).float())
        near = (ties * scale).float()
        for step in (-2, -1, 0, 1, 2):
            v = (near.view(torch.int32) + step).view(torch.float32)
            row = torch.zeros(256)
            row[:126], row[127] = v, m
            row[128:128 + 126], row[255] = -v, m
            rows.append(row)
    x = torch.stack(rows)
    q, scale = plain_fp8(x)
    out = ops.fp8_rows(*x.shape, DEV)
    ops.quantize_fp8(x.to(DEV), out)
    assert torch.equal(out.scale.cpu(), scale) and torch.equal(out.data.cpu().double(), q)


def test_quantise_rows_that_8_bits_cannot_say(ops):
    x = rnd(8, 300)
    x[0] = 0
    x[1, 5], x[2, 290], x[3, 128], x[4, 0] = math.inf, -math.inf, math.nan, 1e-42
    x[5] = 2.0 ** -110
    x[6, 256:] = 3.4e38
    x[7] = -0.0
    q, scale = plain_fp8(x)
    out = ops.fp8_rows(8, 300, DEV)
    ops.quantize_fp8(x.to(DEV), out)
    same = (out.scale.cpu() == scale) | (out.scale.cpu().isnan() & scale.isnan())
    assert same.all() and torch.equal(out.data.cpu().double(), q)
    values = ops.fp8_values(out, torch.empty((8, 300), device=DEV)).cpu()
    assert values[1, :128].isnan().all() and values[1, 128:].isfinite().all() and values[2, 256:].isnan().all() and values[3, 128:256].isnan().all()


def test_rows_of_other_strides_and_slices(ops):
    wide = rnd(9, 700).to(torch.bfloat16)
    q, scale = plain_fp8(wide[:, 3:503].float())
    room = ops.fp8_rows(12, 500, DEV)
    ops.quantize_fp8(wide.to(DEV)[:, 3:503], room[2:11])
    assert torch.equal(room.data[2:11].cpu().double(), q) and torch.equal(room.scale[2:11].cpu(), scale)
    out = torch.full((9, 601), 7.0, device=DEV)
    ops.fp8_values(room[2:11], out[:, 1:501])
    assert torch.equal(out[:, 1:501].cpu(), values_of(q, scale).float()) and (out[:, 501:] == 7).all() and (out[:, 0] == 7).all()


# ---- products in 8 bits ----

CUTS = [16111, 16121, 32111, 64111, 128211]


def run_product(ops, rows, n, k, *, bias=None, accumulate=False, glu=False, dtype=torch.float32, cut=0, seed=0):
    q, sq = plain_fp8(rnd(rows, k, seed=seed) * torch.exp(rnd(rows, 1, seed=5)))
    wq, ws = fp8_weight(n, k, seed)
    a, w = values_of(q, sq), weight_values(wq, ws)
    want, slack = a @ w.T, product_slack(a, w, -(-k // 128))
    width = n
    if glu:
        want, slack = units_and_slack(want, slack)
        width = n // 2
    if bias is not None:
        want = want + bias.double()
        slack = slack + ULP * want.abs()
    before = rnd(rows, width, seed=9).to(dtype)
    if accumulate is True:
        want = want + before.double()
        slack = slack + ULP * want.abs()
    if accumulate == ops.EPILOGUE_RELU2 and accumulate is not True and accumulate is not False:
        slack = (2 * want.abs() + slack) * slack + ULP * want ** 2
        want = want.clamp(min=0) ** 2
    out = torch.full((rows + 2, width + 5), 3.0, dtype=dtype, device=DEV)
    view = out[1:rows + 1, 2:width + 2] if (n + k) % 2 else out[1:rows + 1, :width]
    view.copy_(before)
    ops.gemm_fp8(rows_of(ops, q, sq), ops.pack_fp8(wq.to(DEV), ws.to(DEV), glu=glu), view, None if bias is None else bias.to(DEV), accumulate,
                 swiglu="silu" if glu else False, cut=cut)
    check(view, want, slack, dtype, f"{rows} x {n} x {k} cut {cut}")
    view.fill_(3.0)
    assert (out == 3.0).all()
    return want


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 128, 128), (3, 130, 129), (16, 64, 512), (17, 1003, 300), (33, 256, 640), (64, 384, 1000), (65, 129, 2049),
                                      (128, 512, 256), (129, 255, 385), (300, 700, 900), (1, 4096, 4096), (8, 2048, 12288)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product(ops, rows, n, k, dtype):
    run_product(ops, rows, n, k, dtype=dtype)


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("rows,n,k", [(5, 300, 700), (40, 129, 1100), (150, 700, 520), (1, 128, 2000)])
def test_product_of_every_cut(ops, rows, n, k, cut):
    run_product(ops, rows, n, k, cut=cut)
    run_product(ops, rows, 16 * (n // 16), k, glu=True, dtype=torch.bfloat16, cut=cut)


@pytest.mark.parametrize("nt", [16, 32])
@pytest.mark.parametrize("blocks", [2, 3, 4, 5, 8])
def test_product_of_clusters(ops, nt, blocks):
    for rows in sorted({1, 8, 9, nt - 1, nt, nt + 1, 3 * nt}):
        run_product(ops, rows, 260, 1930, cut=nt * 1000 + 110 + blocks, seed=blocks)
        run_product(ops, rows, 272, 1800, glu=True, dtype=torch.bfloat16, cut=nt * 1000 + 110 + blocks, seed=rows)


@pytest.mark.parametrize("cut", [128212, 128214])
@pytest.mark.parametrize("rows,n,k", [(1, 100, 520), (31, 300, 700), (128, 256, 1024), (129, 384, 2049), (300, 129, 640), (97, 1003, 1930)])
def test_product_of_wide_clusters(ops, rows, n, k, cut):
    run_product(ops, rows, n, k, cut=cut, bias=rnd(n, seed=4))
    run_product(ops, rows, n, k, cut=cut, accumulate=True, dtype=torch.bfloat16)
    run_product(ops, rows, 16 * (n // 16), k, glu=True, cut=cut)
    run_product(ops, rows, 16 * (n // 16), k, glu=True, dtype=torch.bfloat16, cut=cut)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(3, 200, 260), (70, 333, 500)])
def test_epilogues(ops, rows, n, k, dtype):
    bias = rnd(n, seed=4)
    run_product(ops, rows, n, k, bias=bias, dtype=dtype)
    run_product(ops, rows, n, k, bias=bias.to(torch.bfloat16), accumulate=True, dtype=dtype)
    run_product(ops, rows, n, k, accumulate=True, dtype=dtype)
    run_product(ops, rows, n, k, bias=bias, accumulate=ops.EPILOGUE_RELU2, dtype=dtype)


@pytest.mark.parametrize("hidden", [8, 72, 128, 136, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_units(ops, hidden, dtype):
    for rows in (1, 20, 140):
        run_product(ops, rows, 2 * hidden, 400, glu=True, dtype=dtype)


def test_product_takes_over_what_is_not_a_number(ops):
    x = rnd(4, 300)
    x[2, 130] = math.inf
    rows8 = ops.fp8_rows(4, 300, DEV)
    ops.quantize_fp8(x.to(DEV), rows8)
    wq, ws = fp8_weight(200, 300)
    out = torch.empty((4, 200), device=DEV)
    ops.gemm_fp8(rows8, ops.pack_fp8(wq.to(DEV), ws.to(DEV)), out, accumulate=ops.EPILOGUE_RELU2)
    assert out[2].isnan().all() and out[[0, 1, 3]].isfinite().all()


def test_empty_product(ops):
    wq, ws = fp8_weight(200, 300)
    ops.gemm_fp8(ops.fp8_rows(0, 300, DEV), ops.pack_fp8(wq.to(DEV), ws.to(DEV)), torch.empty((0, 200), device=DEV))


# ---- groups ----

def plain_groups(choice, groups):
    flat = choice.flatten().tolist()
    order = [p for g in range(groups) for p in range(len(flat)) if flat[p] == g] if len(flat) < 3000 else None
    if order is None:
        key = torch.tensor([c if 0 <= c < groups else groups for c in flat])
        order = torch.sort(key, stable=True).indices[:int((key < groups).sum())].tolist()
    offsets = [0]
    for n in torch.bincount(torch.tensor([c for c in flat if 0 <= c < groups], dtype=torch.long), minlength=groups).tolist():
        offsets.append(offsets[-1] + n)
    place = [-1] * len(flat)
    for i, p in enumerate(order):
        place[p] = i
    return offsets, order + [-1] * (len(flat) - len(order)), place


def choices(rows, top, groups, seed=0, unused=0.2, few=None):
    g = gen(seed + rows + 31 * groups)
    score = torch.rand((rows, groups), generator=g)
    if few:
        score[:, few:] -= 2
    choice = score.topk(top, dim=1).indices.to(torch.int32)
    choice[torch.rand((rows,), generator=g) < unused] = -1
    return choice


@pytest.mark.parametrize("rows,top,groups", [(0, 2, 4), (1, 1, 1), (1, 8, 128), (3, 2, 1024), (31, 1, 5), (8, 8, 128), (128, 8, 7 + 1), (300, 4, 60), (1025, 3, 33), (4096, 8, 256),
                                             (16384, 8, 256), (20011, 5, 1000), (70001, 4, 300)])
def test_group_rows(ops, rows, top, groups):
    choice = choices(rows, top, groups) if rows else torch.empty((0, top), dtype=torch.int32)
    if rows > 20:
        choice[7, 0] = groups              # outside: nobody
        choice[9, top - 1] = -2 ** 31
    room = ops.row_groups(rows, top, groups, DEV)
    for _ in range(2):
        ops.group_rows(choice.to(DEV), room)
        offsets, order, place = plain_groups(choice, groups)
        assert room.offsets.tolist() == offsets and room.order.tolist() == order and room.place.flatten().tolist() == place


def test_group_rows_of_one_expert_and_of_none(ops):
    room = ops.row_groups(5000, 2, 9, DEV)
    for choice in (torch.full((5000, 2), 8, dtype=torch.int32), torch.full((5000, 2), -1, dtype=torch.int32), torch.zeros((5000, 2), dtype=torch.int32)):
        ops.group_rows(choice.to(DEV), room)
        offsets, order, place = plain_groups(choice, 9)
        assert room.offsets.tolist() == offsets and room.order.tolist() == order and room.place.flatten().tolist() == place
    wide = torch.full((40, 7), 99, dtype=torch.int32)
    wide[:, 2:4] = choices(40, 2, 9)
    ops.group_rows(wide.to(DEV)[:, 2:4], room.first(40))
    offsets, order, place = plain_groups(wide[:, 2:4], 9)
    assert room.offsets.tolist() == offsets and room.order[:80].tolist() == order and room.place[:40].flatten().tolist() == place


# ---- products of groups ----

def run_grouped(ops, kind, choice, groups, n, k, *, glu=False, dtype=torch.float32, by_pair=False, cut=0, seed=0):
    rows, top = choice.shape
    pairs, width = rows * top, n // 2 if glu else n
    room = ops.row_groups(rows, top, groups, DEV)
    ops.group_rows(choice.to(DEV), room)
    offsets, order, _ = plain_groups(choice, groups)
    m = pairs if by_pair else rows
    x = rnd(m, k, seed=seed) * torch.exp(rnd(m, 1, seed=5))
    if kind == "fp8":
        q, sq = plain_fp8(x)
        a, av = rows_of(ops, q, sq), values_of(q, sq)
        weights = [fp8_weight(n, k, seed + g) for g in range(groups)]
        packed = ops.pack_fp8(torch.stack([w[0] for w in weights]).to(DEV), torch.stack([w[1] for w in weights]).to(DEV), glu=glu)
        wv = [weight_values(*w) for w in weights]
    else:
        held = torch.zeros((m, -(-k // 8) * 8 + 8), dtype=torch.bfloat16, device=DEV)
        held[:, :k] = x.to(torch.bfloat16).to(DEV)
        a, av = held[:, :k], x.to(torch.bfloat16).double()
        weights = torch.stack([rnd(n, k, seed=seed + g) / math.sqrt(k) for g in range(groups)]).to(torch.bfloat16)
        packed = ops.pack_grouped(weights.to(DEV), glu=glu)
        wv = weights.double()
    out = torch.full((pairs, width + (3 if n % 2 else 8)), 5.0, dtype=dtype, device=DEV)
    ops.gemm_grouped(a, packed, room, out[:, :width], swiglu="silu" if glu else False, by_pair=by_pair, cut=cut)
    for g in range(groups):
        lo, hi = offsets[g], offsets[g + 1]
        if lo == hi:
            continue
        rows_g = av[lo:hi] if by_pair else av[[p // top for p in order[lo:hi]]]
        want = rows_g @ wv[g].T
        slack = product_slack(rows_g, wv[g], -(-k // 64)) if kind == "fp8" else (k + 4) * ULP * (rows_g.abs() @ wv[g].abs().T)
        if glu:
            want, slack = units_and_slack(want, slack)
        check(out[lo:hi, :width], want, slack, dtype, f"{kind} group {g} of {groups} ({hi - lo} pairs) cut {cut}")
    assert (out[offsets[-1]:] == 5.0).all() and (out[:, width:] == 5.0).all()
    return out[:, :width], room


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("rows,top,groups,n,k", [(1, 1, 1, 8, 8), (1, 8, 16, 256, 512), (3, 2, 7, 130, 136), (8, 4, 40, 400, 1000), (60, 3, 5, 257, 520), (200, 2, 3, 384, 264),
                                                 (500, 4, 6, 200, 328)])
@pytest.mark.parametrize("by_pair", [False, True])
def test_grouped(ops, kind, rows, top, groups, n, k, by_pair):
    choice = choices(rows, top, groups)
    run_grouped(ops, kind, choice, groups, n, k, by_pair=by_pair)
    run_grouped(ops, kind, choice, groups, 16 * (n // 16) + 16, k, glu=True, dtype=torch.bfloat16, by_pair=by_pair)


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("by_pair", [False, True])
def test_grouped_of_every_cut(ops, kind, cut, by_pair):
    run_grouped(ops, kind, choices(90, 3, 6, few=4), 6, 300, 1000, cut=cut, by_pair=by_pair)
    run_grouped(ops, kind, choices(90, 3, 6, few=4), 6, 272, 264, glu=True, cut=cut, by_pair=by_pair)


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
def test_groups_of_all_lengths(ops, kind):
    """0, 1 and up to 300 pairs of one group, beside groups that nobody asks."""
    counts = [0, 1, 15, 16, 17, 0, 127, 128, 129, 300, 2, 0]
    choice = torch.cat([torch.full((c, 1), g, dtype=torch.int32) for g, c in enumerate(counts)])
    choice = choice[torch.randperm(len(choice), generator=gen(1))]
    run_grouped(ops, kind, choice, len(counts), 140, 200)
    run_grouped(ops, kind, torch.full((9, 2), -1, dtype=torch.int32), 3, 140, 200)          # nobody asks anybody


def test_many_groups(ops):
    run_grouped(ops, "bfloat16", choices(40, 2, 1024), 1024, 16, 16)


def test_grouped_of_unfilled_groups_writes_nothing(ops):
    room = ops.row_groups(4, 2, 3, DEV)
    packed = ops.pack_grouped(rnd(3, 16, 8).to(torch.bfloat16).to(DEV))
    out = torch.full((8, 16), 5.0, device=DEV)
    ops.gemm_grouped(torch.ones((4, 8), dtype=torch.bfloat16, device=DEV), packed, room, out)
    assert (out == 5).all()


# ---- the sum of the answers ----

@pytest.mark.parametrize("rows,top,dim", [(1, 1, 1), (5, 2, 7), (30, 8, 256), (9, 5, 1000), (700, 4, 513), (64, 9, 2048)])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_combine(ops, rows, top, dim, types, accumulate):
    groups = max(top, 11)
    choice = choices(rows, top, groups)
    choice[rows // 2, 0] = -1
    room = ops.row_groups(rows, top, groups, DEV)
    ops.group_rows(choice.to(DEV), room)
    offsets, _, place = plain_groups(choice, groups)
    answers = rnd(rows * top, dim).to(types[0])
    answers[offsets[-1]:] = math.nan                  # (behind the last pair: nobody's)
    share = rnd(rows, top, seed=2)
    share[choice < 0] = math.nan                      # (of a choice that asks nobody)
    before = rnd(rows, dim, seed=8).to(types[1])
    out = before.to(DEV)
    ops.combine_groups(answers.to(DEV), room, share.to(DEV), out, accumulate=accumulate)
    place = torch.tensor(place).view(rows, top)
    want, size = torch.zeros((rows, dim), dtype=torch.float64), torch.zeros((rows, dim), dtype=torch.float64)
    for c in range(top):
        there = place[:, c] >= 0
        one = answers[place[there, c]].double() * share[there, c].double()[:, None]
        want[there] += one
        size[there] += one.abs()
    if accumulate:
        want, size = want + before.double(), size + before.double().abs()
    check(out, want, (top + 1) * ULP * size, types[1])


# ---- together ----

@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("rows", [1, 16, 200])
def test_a_layer_of_experts(ops, kind, rows):
    """What a served layer calls: against 64 bits with the same two roundings in between (rows and units to the products' type)."""
    top, groups, dim, hidden = 4, 12, 256, 136
    choice, share = choices(rows, top, groups, unused=0.1), torch.softmax(rnd(rows, top, seed=2), dim=1)
    x = rnd(rows, dim).to(torch.bfloat16)
    gu, dn = rnd(groups, 2 * hidden, dim) / math.sqrt(dim), rnd(groups, dim, hidden, seed=1) / math.sqrt(hidden)
    make = ops.quantize_weight_fp8 if kind == "fp8" else lambda w, glu=False: ops.pack_grouped(w.to(torch.bfloat16), glu)
    gate_up, down = make(gu.to(DEV), glu=True), make(dn.to(DEV))
    if kind == "fp8":          # (the values that the packed weights stand for)
        def plain(w):
            return torch.stack([weight_values(*(lambda b: (b[0], b[1]))(plain_weight(one))) for one in w])
        guv, dnv = plain(gu), plain(dn)
    else:
        guv, dnv = gu.to(torch.bfloat16).double(), dn.to(torch.bfloat16).double()
    room = ops.row_groups(rows, top, groups, DEV)
    units = torch.empty((rows * top, hidden), dtype=torch.float32 if kind == "fp8" else torch.bfloat16, device=DEV)
    answers, out = torch.empty((rows * top, dim), device=DEV), torch.full((rows, dim), 2.0, device=DEV)

    def layer():
        a = x.to(DEV)
        ops.group_rows(choice.to(DEV), room)
        if kind == "fp8":
            a8, u8 = ops.fp8_rows(rows, dim, DEV), ops.fp8_rows(rows * top, hidden, DEV)
            ops.quantize_fp8(a, a8)
            a = a8
        ops.gemm_grouped(a, gate_up, room, units, swiglu="silu")
        u = units
        if kind == "fp8":
            ops.quantize_fp8(units, u8)
            u = u8
        ops.gemm_grouped(u, down, room, answers, by_pair=True)
        ops.combine_groups(answers, room, share.to(DEV), out, accumulate=True)
    layer()
    xv = values_of(*plain_fp8(x.float())) if kind == "fp8" else x.double()
    want = torch.full((rows, dim), 2.0, dtype=torch.float64)
    for r in range(rows):
        for c in range(top):
            e = int(choice[r, c])
            if e < 0:
                continue
            gate, up = (guv[e] @ xv[r]).chunk(2)
            u = (gate * torch.sigmoid(gate) * up)[None]
            u = values_of(*plain_fp8(u.float())) if kind == "fp8" else u.to(torch.bfloat16).double()
            want[r] += float(share[r, c]) * (dnv[e] @ u[0])
    # a unit next to a tie may fall to the other side: a step of its type (2^-3 or 2^-8 of it) in one unit of some hundreds
    step = 2.0 ** -3 if kind == "fp8" else 2.0 ** -8
    size = (want - 2.0).abs().amax(dim=1, keepdim=True).clamp(min=0.1)
    off = (out.cpu().double() - want).abs()
    assert (off <= step * size).all() and float((off / size).mean()) < (2e-3 if kind == "fp8" else 2e-5)


def plain_weight(w):
    """(q, scale) of a weight rounded in blocks of 128 x 128, as `quantize_weight_fp8` says it."""
    n, k = w.shape
    padded = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128))
    blocks = padded.view(padded.shape[0] // 128, 128, -1, 128)
    scale = (blocks.abs().amax(dim=(1, 3)).clamp(min=2.0 ** -100) / 448.0)
    q = plain_e4m3((blocks / scale[:, None, :, None]).double()).reshape(padded.shape)[:n, :k]
    return q, scale
