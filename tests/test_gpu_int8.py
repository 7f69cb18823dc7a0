"""The linears in 8-bit integers, each operator alone (GPU): against plain forms whose every rounding is the kernels' own (equal bits),
and against the definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    return o


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + 7 * sum(shape)))


def plain_int8(v):
    """(q, scale) of the float32 rows of v, on the CPU: IEEE float32 operations, half to even."""
    m = v.abs().amax(dim=1)
    inverse = torch.where(m < 2.0 ** -100, torch.zeros_like(m), torch.tensor(127.0) / m)
    scale = torch.where(m < 2.0 ** -100, torch.zeros_like(m), m / 127.0)
    bad = ~torch.isfinite(v).all(dim=1)
    q = torch.round(v * inverse[:, None]).clamp(-127, 127)
    q[bad], scale[bad] = 0.0, float("nan")
    q[m < 2.0 ** -100] = 0.0
    return q.to(torch.int8), scale


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))


WIDTHS = [1, 2, 3, 8, 15, 16, 17, 100, 128, 255, 1000, 1024, 1027, 2048, 4096, 5120, 8191, 12288, 17408, 24580]


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_gives_the_plain_bits(ops, dim, rows, dtype):
    x = (rnd(rows, dim) * torch.exp(rnd(rows, 1, seed=3))).to(dtype)
    want_q, want_scale = plain_int8(x.float())
    out = ops.int8_rows(rows, dim, DEV)
    ops.quantize_int8(x.to(DEV), out)
    assert torch.equal(out.data.cpu(), want_q) and torch.equal(out.scale.cpu(), want_scale)
    for kind in (torch.float32, torch.bfloat16):
        values = ops.int8_values(out, torch.empty(rows, dim, dtype=kind, device=DEV))
        assert torch.equal(values.cpu(), (want_q.float() * want_scale[:, None]).to(kind))


@pytest.mark.parametrize("rows", [2, 63, 64, 147, 148, 300, 2500])
@pytest.mark.parametrize("dim", [64, 257, 4096])
def test_quantize_of_many_rows(ops, rows, dim):
    x = rnd(rows, dim)
    x[rows // 2] = 0.0
    want_q, want_scale = plain_int8(x)
    out = ops.int8_rows(rows, dim, DEV)
    ops.quantize_int8(x.to(DEV), out)
    assert torch.equal(out.data.cpu(), want_q) and torch.equal(out.scale.cpu(), want_scale)


def test_quantize_rows_that_8_bits_cannot_say(ops):
    dim = 513
    x = rnd(9, dim)
    x[0] = 0.0                                    # zeros
    x[1], x[1, 5] = 0.0, 1e-42                    # less than 127 / m has in float32
    x[2, 7] = math.inf
    x[3, 512] = -math.inf
    x[4, 0] = math.nan
    x[5, 511], x[5, 3] = math.nan, math.inf
    x[6, 100] = 3.4e38                            # one value beside which the others vanish
    x[7] = torch.where(torch.arange(dim) % 2 == 0, 63.5, -127.0)        # halves: to even
    x[8] = 2.0 ** -100                            # the smallest row that is not zeros
    want_q, want_scale = plain_int8(x)
    assert want_q[8].eq(127).all() and want_q[7, 0] == 64 and want_q[:6, 1].tolist()[:2] == [0, 0]
    for dtype in (torch.float32, torch.bfloat16):
        rows = x.to(dtype)
        q, scale = plain_int8(rows.float())
        out = ops.int8_rows(9, dim, DEV)
        ops.quantize_int8(rows.to(DEV), out)
        assert torch.equal(out.data.cpu(), q) and same(out.scale.cpu(), scale)
        assert torch.isnan(out.scale[2:6]).all()


def test_quantize_reads_strided_rows_and_writes_its_own_only(ops):
    wide = rnd(7, 400).to(DEV)
    x = wide[:, 33:233]                           # a view that begins at an odd 4 bytes
    room = torch.full((7, 256), 77, dtype=torch.int8, device=DEV)
    scale = torch.full((9,), 5.0, device=DEV)
    ops.quantize_int8(x, ops.Int8Rows(room[:, :200], scale[1:8]))
    q, s = plain_int8(x.cpu())
    assert torch.equal(room[:, :200].cpu(), q) and torch.equal(scale[1:8].cpu(), s)
    assert room[:, 200:].eq(77).all() and scale[0] == 5 and scale[8] == 5
    ops.quantize_int8(x[:0], ops.int8_rows(0, 200, DEV))          # no rows


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("add", [None, torch.float32, torch.bfloat16])
def test_add_rmsnorm(ops, dim, add):
    rows, eps = 4, 1e-5
    x = rnd(rows, dim) * 3
    y = None if add is None else rnd(rows, dim, seed=1).to(add)
    for gain_dtype in (torch.float32, torch.bfloat16):
        gain = (1 + 0.3 * rnd(dim, seed=2)).to(gain_dtype)
        out, total = ops.int8_rows(rows, dim, DEV), torch.empty(rows, dim, device=DEV)
        dev = x.to(DEV)
        ops.add_rmsnorm_int8(dev, gain.to(DEV), eps, out, y=None if y is None else y.to(DEV), total=None if y is None else total)
        t = x if y is None else x + y.float()
        if y is not None:
            assert torch.equal(total.cpu(), t) and torch.equal(dev.cpu(), x)
        check_norm(out, t, gain, eps, dim)
        if y is not None:                        # in place
            again = ops.int8_rows(rows, dim, DEV)
            ops.add_rmsnorm_int8(dev, gain.to(DEV), eps, again, y=y.to(DEV))
            assert torch.equal(dev.cpu(), t) and torch.equal(again.data, out.data) and torch.equal(again.scale, out.scale)


def check_norm(out, t, gain, eps, dim):
    """Against 64 bits. The mean's relative error: a thread's sum is a chain of at most dim / 32 + 4 fused multiply-adds, ten more of
    the reduction behind it, each within 2^-24 (the squares are positive), half of it in the root; two products and the divisions
    behind that, 2^-24 each. A quotient v / scale is at most 127, so that error moves it by 127 times as much."""
    t64 = t.double()
    v = t64 / torch.sqrt((t64 ** 2).mean(dim=1, keepdim=True) + eps) * gain.double()
    off = (0.5 * (dim / 32 + 14) + 6) * 2.0 ** -24
    scale = v.abs().amax(dim=1) / 127
    got = out.scale.cpu().double()
    assert ((got - scale).abs() <= off * scale).all()
    q = out.data.cpu().double()
    assert ((v / scale[:, None] - q).abs() <= 0.5 + 127 * 2 * off).all() and q.abs().amax(dim=1).eq(127).all()


@pytest.mark.parametrize("rows", [1, 2, 63, 149, 1000])
@pytest.mark.parametrize("dim", [96, 1030, 4096])
def test_add_rmsnorm_of_many_rows(ops, rows, dim):
    x, y, gain = rnd(rows, dim), rnd(rows, dim, seed=1).to(torch.bfloat16), 1 + 0.3 * rnd(dim, seed=2)
    out, total = ops.int8_rows(rows, dim, DEV), torch.empty(rows, dim, device=DEV)
    ops.add_rmsnorm_int8(x.to(DEV), gain.to(DEV), 1e-6, out, y=y.to(DEV), total=total)
    assert torch.equal(total.cpu(), x + y.float())
    check_norm(out, x + y.float(), gain, 1e-6, dim)
    one = ops.int8_rows(1, dim, DEV)              # a row alone has the same bits
    ops.add_rmsnorm_int8(x[rows - 1:].to(DEV), gain.to(DEV), 1e-6, one, y=y[rows - 1:].to(DEV))
    assert torch.equal(one.data[0], out.data[rows - 1]) and one.scale[0] == out.scale[rows - 1]


def test_add_rmsnorm_odd_rows(ops):
    dim = 260
    x, y, gain = rnd(6, dim), rnd(6, dim, seed=1), 1 + 0.3 * rnd(dim, seed=2)
    x[0], y[0] = 0.0, 0.0
    x[1, 3] = math.inf
    y[2, 259] = math.nan
    x[3] *= 1e30                                  # the squares leave float32
    x[4], y[4] = 1e-30, 0.0                       # far below eps
    out = ops.int8_rows(6, dim, DEV)
    dev = x.to(DEV)
    ops.add_rmsnorm_int8(dev, gain.to(DEV), 1e-6, out, y=y.to(DEV))
    assert same(dev.cpu(), x + y)
    scale = out.scale.cpu()
    assert scale[0] == 0 and out.data[0].eq(0).all()
    assert torch.isnan(scale[1]) and torch.isnan(scale[2]) and out.data[1:3].eq(0).all()
    check_norm(out[3:], (x + y)[3:], gain, 1e-6, dim)
    small = ops.int8_rows(3, dim, DEV)            # ... or vanish in it, without an eps
    ops.add_rmsnorm_int8((x[3:] * torch.tensor([[1e-55], [1.0], [1e-22]])).to(DEV), gain.to(DEV), 0.0, small)
    # (1e-55 is zero in float32: a row of zeros without an eps is 0 / 0, not a number)
    assert torch.isnan(small.scale[0]) and small.data[0].eq(0).all()
    check_norm(small[1:], (x[3:] * torch.tensor([[1e-55], [1.0], [1e-22]]))[1:], gain, 0.0, dim)
    # strided rows, and memory beside them left alone
    xs, ys, ts = (torch.full((6, 300), 9.0, device=DEV) for _ in range(3))
    xs[:, 4:4 + dim], ys[:, 1:1 + dim] = x.to(DEV), y.to(DEV)
    again = ops.int8_rows(6, dim, DEV)
    ops.add_rmsnorm_int8(xs[:, 4:4 + dim], gain.to(DEV), 1e-6, again, y=ys[:, 1:1 + dim], total=ts[:, 3:3 + dim])
    assert torch.equal(again.data, out.data) and same(again.scale, out.scale)
    assert same(ts[:, 3:3 + dim].cpu(), x + y) and ts[:, :3].eq(9).all() and ts[:, 3 + dim:].eq(9).all()


# ---- the product ----------------------------------------------------------------------------------------------------

def integers(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8)
    return q, torch.rand((rows,), generator=g) * 0.02 + 1e-3


def on_gpu(ops, q, scale):
    rows8 = ops.int8_rows(q.shape[0], q.shape[1], DEV)
    rows8.data.copy_(q)
    rows8.scale.copy_(scale)
    return rows8


def plain_product(a, sa, w, sw, bias=None, old=None, relu2=False):
    """Float32 with the kernels' roundings: the sum (exact in 64 bits) rounded once, then token scale, weight scale, bias, old value."""
    v = (a.to(DEV).double() @ w.to(DEV).double().T).cpu().float() * sa[:, None] * sw[None, :]
    if bias is not None:
        v = v + bias.float()
    if relu2:
        v = v.clamp(min=0) * v.clamp(min=0)
    return v if old is None else v + old.float()


ROWS = [1, 2, 8, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 161, 200, 255, 256, 257, 300, 384, 511, 513, 700]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("width,dim", [(256, 512), (1003, 2049), (129, 17), (384, 4096)])
def test_product_gives_the_plain_bits(ops, rows, width, dim):
    (a, sa), (w, sw) = integers(rows, dim, rows), integers(width, dim, width)
    a8, packed = on_gpu(ops, a, sa), ops.pack_int8(w.to(DEV), sw.to(DEV))
    want = plain_product(a, sa, w, sw)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.empty(rows, width, dtype=dtype, device=DEV)
        ops.gemm_int8(a8, packed, out)
        ops.check_kernel_errors()
        assert torch.equal(out.cpu(), want.to(dtype))


@pytest.mark.parametrize("rows,width,dim", [(1, 1, 1), (3, 1, 5), (1, 7, 15), (2, 16, 16), (40, 128, 127), (130, 3, 128), (260, 40, 129), (300, 31, 1000),
                                            (600, 65, 31), (1, 4096, 12288), (8, 6144, 4096), (64, 4096, 1024), (16, 151, 20000), (600, 2048, 640),
                                            (5, 30000, 64), (2048, 512, 384), (4100, 300, 200)])
def test_product_sizes(ops, rows, width, dim):
    (a, sa), (w, sw) = integers(rows, dim, 1), integers(width, dim, 2)
    out = torch.empty(rows, width, device=DEV)
    ops.gemm_int8(on_gpu(ops, a, sa), ops.pack_int8(w.to(DEV), sw.to(DEV)), out)
    ops.check_kernel_errors()
    assert torch.equal(out.cpu(), plain_product(a, sa, w, sw))


def test_product_of_the_largest_sums(ops):
    """-128 * -128 at the longest k: the sum is just below 2^31."""
    K = ops.INT8_MAX_K
    for rows in (3, 300):
        a = torch.full((rows, K), -128, dtype=torch.int8)
        w = torch.full((2, K), -128, dtype=torch.int8)
        w[1] = 127
        out = torch.empty(rows, 2, device=DEV)
        ones = torch.ones(rows), torch.ones(2)
        ops.gemm_int8(on_gpu(ops, a, ones[0]), ops.pack_int8(w.to(DEV), ones[1].to(DEV)), out)
        ops.check_kernel_errors()
        assert out[:, 0].eq(float(K * 128 * 128)).all() and out[:, 1].eq(float(torch.tensor(-K * 128 * 127).float())).all()


@pytest.mark.parametrize("rows", [1, 16, 40, 130, 256, 300, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias_dtype", [None, torch.float32, torch.bfloat16])
def test_product_epilogues(ops, rows, dtype, bias_dtype):
    width, dim = 530, 400
    (a, sa), (w, sw) = integers(rows, dim, 3), integers(width, dim, 4)
    a8, packed = on_gpu(ops, a, sa), ops.pack_int8(w.to(DEV), sw.to(DEV))
    bias = None if bias_dtype is None else rnd(width).to(bias_dtype)
    b = None if bias is None else bias.to(DEV)
    for pad in (0, 1, 6):                          # rows of the result that begin anywhere
        room = torch.full((rows, width + 2 * pad), 4.0, dtype=dtype, device=DEV)
        out = room[:, pad:pad + width]
        ops.gemm_int8(a8, packed, out, b)
        assert torch.equal(out.cpu(), plain_product(a, sa, w, sw, bias).to(dtype))
        old = rnd(rows, width, seed=5).to(dtype)
        out.copy_(old)
        ops.gemm_int8(a8, packed, out, b, accumulate=True)
        assert torch.equal(out.cpu(), plain_product(a, sa, w, sw, bias, old).to(dtype))
        ops.gemm_int8(a8, packed, out, b, accumulate=ops.EPILOGUE_RELU2)
        assert torch.equal(out.cpu(), plain_product(a, sa, w, sw, bias, relu2=True).to(dtype))
        assert room[:, :pad].eq(4).all() and room[:, pad + width:].eq(4).all()
    ops.check_kernel_errors()


@pytest.mark.parametrize("rows", [1, 16, 40, 130, 256, 300, 700])
@pytest.mark.parametrize("hidden", [8, 200, 264, 1024])
@pytest.mark.parametrize("kind", ["silu", "gelu_tanh", "swish_clamped"])
def test_product_gated(ops, rows, hidden, kind):
    dim = 272
    (a, sa), (w, sw) = integers(rows, dim, 3), integers(2 * hidden, dim, 4)
    sw = sw * 0.15                                 # gates of a few units
    a8, packed = on_gpu(ops, a, sa), ops.pack_int8(w.to(DEV), sw.to(DEV), glu=True)
    both = plain_product(a, sa, w, sw).double()
    g, u = both[:, :hidden], both[:, hidden:]
    assert float(g.abs().max()) < 40
    if kind == "silu":
        want = g * torch.sigmoid(g) * u
    elif kind == "gelu_tanh":
        want = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    else:
        g = g.clamp(max=3.0)
        want = g * torch.sigmoid(1.702 * g) * (u.clamp(-3.0, 3.0) + 1)
    word = ops.glu_descriptor(kind, 3.0)
    for dtype, pad in ((torch.float32, 0), (torch.bfloat16, 0), (torch.bfloat16, 3)):
        room = torch.full((rows, hidden + pad), 4.0, dtype=dtype, device=DEV)
        ops.gemm_int8(a8, packed, room[:, pad:], swiglu=word)
        # the activation's exponential: its argument (up to 64 for silu and the clamped unit, the cube's for GELU, whose factor is then
        # 0 or 1) rounded to 2^-24 of itself, base-2 exponential and quotient within 2^-21; two products: below 2^-16 of the value, and
        # an absolute rest where the exponential leaves float32
        rel = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -8
        assert torch.allclose(room[:, pad:].cpu().double(), want, rtol=rel, atol=1e-6 * float(want.abs().max()))
        assert room[:, :pad].eq(4).all()
    ops.check_kernel_errors()


@pytest.mark.parametrize("cut,rows,width,dim", [
    (1, 1, 128, 128), (11, 256, 300, 1300), (2, 3, 200, 300), (3, 17, 129, 1000), (4, 40, 1003, 2049), (15, 200, 70, 900), (16, 256, 260, 4096),
    (17, 100, 256, 1025), (18, 256, 400, 3000), (8, 8, 384, 8192), (8, 1, 100, 1024), (11, 1, 700, 4096), (11, 256, 129, 500), (12, 40, 1003, 2049),
    (13, 64, 400, 2500), (14, 250, 130, 3000), (16, 16, 384, 8192), (18, 256, 200, 1024), (18, 7, 1400, 2300), (2, 144, 300, 256), (12, 160, 129, 129),
    (7, 24, 64, 12000),
    # groups of tokens: even ones, a short last one, fewer than were asked for, one token in the last
    (201, 32, 10, 20), (202, 130, 250, 700), (211, 300, 2600, 513), (301, 257, 129, 500), (312, 700, 400, 333), (401, 777, 1003, 2049),
    (512, 513, 700, 1111), (812, 2048, 3000, 256), (911, 2100, 5000, 300), (713, 100, 300, 900), (1201, 777, 1003, 2049), (3002, 500, 257, 640),
    (1001, 161, 128, 200), (218, 500, 130, 1500), (1712, 4100, 130, 300)])
def test_product_cut_up(ops, cut, rows, width, dim):
    """Every way of cutting the work gives the same bits."""
    (a, sa), (w, sw) = integers(rows, dim, 11), integers(width, dim, 12)
    bias, old = rnd(width), rnd(rows, width, seed=5)
    a8, packed = on_gpu(ops, a, sa), ops.pack_int8(w.to(DEV), sw.to(DEV))
    for _ in range(3):
        out = old.to(DEV)
        ops.gemm_int8(a8, packed, out, bias.to(DEV), accumulate=True, cut=cut)
        out16 = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
        ops.gemm_int8(a8, packed, out16, cut=cut)
        ops.check_kernel_errors()
        assert torch.equal(out.cpu(), plain_product(a, sa, w, sw, bias, old))
        assert torch.equal(out16.cpu(), plain_product(a, sa, w, sw).to(torch.bfloat16))


def test_a_rows_bits_do_not_depend_on_its_batch(ops):
    """Every kernel and every way of cutting the work: a row alone, in small and in large batches."""
    dim, width = 1111, 2050
    (a, sa), (w, sw) = integers(900, dim, 5), integers(width, dim, 6)
    a8, packed = on_gpu(ops, a, sa), ops.pack_int8(w.to(DEV), sw.to(DEV))
    whole = torch.empty(900, width, device=DEV)
    ops.gemm_int8(a8, packed, whole)
    glu = ops.pack_int8(w[:2048].to(DEV), sw[:2048].to(DEV) * 0.01, glu=True)
    units = torch.empty(900, 1024, device=DEV)
    ops.gemm_int8(a8, glu, units, swiglu="silu")
    for lo, hi in ((0, 1), (899, 900), (10, 17), (100, 140), (200, 330), (500, 756), (300, 700)):
        out, part = torch.empty(hi - lo, width, device=DEV), torch.empty(hi - lo, 1024, device=DEV)
        ops.gemm_int8(a8[lo:hi], packed, out)
        ops.gemm_int8(a8[lo:hi], glu, part, swiglu="silu")
        assert torch.equal(out, whole[lo:hi]) and torch.equal(part, units[lo:hi])
    ops.check_kernel_errors()


def test_product_of_rows_that_are_not_numbers(ops):
    (a, sa), (w, sw) = integers(300, 256, 7), integers(140, 256, 8)
    sa[5] = math.nan
    a[5] = 0
    sw[17] = 0.0
    for rows in (20, 300):
        out = torch.empty(rows, 140, device=DEV)
        ops.gemm_int8(on_gpu(ops, a[:rows], sa[:rows]), ops.pack_int8(w.to(DEV), sw.to(DEV)), out)
        assert torch.isnan(out[5]).all() and torch.isfinite(out[:5]).all() and torch.isfinite(out[6:]).all() and out[6:, 17].eq(0).all()


def test_product_without_rows(ops):
    packed = ops.pack_int8(*(t.to(DEV) for t in integers(40, 32, 1)))
    ops.gemm_int8(ops.int8_rows(0, 32, DEV), packed, torch.empty(0, 40, device=DEV))


def test_operators_on_another_stream(ops):
    """Each launch goes to the current stream, behind what that stream holds."""
    x = rnd(200, 4096).to(DEV)
    gain = torch.ones(4096, device=DEV)
    packed = ops.quantize_weight_int8(rnd(1024, 4096, seed=1).to(DEV))
    want8, want = ops.int8_rows(200, 4096, DEV), torch.empty(200, 1024, device=DEV)
    ops.add_rmsnorm_int8(x, gain, 1e-6, want8)
    ops.gemm_int8(want8, packed, want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late, rows8, out = torch.zeros_like(x), ops.int8_rows(200, 4096, DEV), torch.empty_like(want)
    with torch.cuda.stream(side):
        for _ in range(20):
            late.copy_(x)
            late.mul_(1.0)
        ops.add_rmsnorm_int8(late, gain, 1e-6, rows8)
        ops.gemm_int8(rows8, packed, out)
    side.synchronize()
    assert torch.equal(out, want)


def test_operators_in_a_graph(ops):
    x, y, gain = rnd(9, 1024).to(DEV), rnd(9, 1024, seed=1).to(torch.bfloat16).to(DEV), torch.ones(1024, device=DEV)
    glu, down = ops.quantize_weight_int8(rnd(1536, 1024, seed=2).to(DEV) / 32, glu=True), ops.quantize_weight_int8(rnd(1024, 768, seed=3).to(DEV) / 28)
    rows8, hidden8 = ops.int8_rows(9, 1024, DEV), ops.int8_rows(9, 768, DEV)
    total, hidden, out = torch.empty_like(x), torch.empty(9, 768, dtype=torch.bfloat16, device=DEV), torch.empty(9, 1024, device=DEV)

    def step():
        ops.add_rmsnorm_int8(x, gain, 1e-6, rows8, y=y, total=total)
        ops.gemm_int8(rows8, glu, hidden, swiglu="silu")
        ops.quantize_int8(hidden, hidden8)
        ops.gemm_int8(hidden8, down, out)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    x.copy_(rnd(9, 1024, seed=9))
    graph.replay()
    got = out.clone()
    step()
    assert torch.equal(got, out)
    ops.check_kernel_errors()


@pytest.mark.parametrize("rows,cols", [(1, 1), (128, 128), (129, 127), (300, 500), (16, 1000), (2064, 336)])
def test_packing_on_the_gpu_gives_the_layout(ops, rows, cols):
    (w, scale) = integers(rows, cols + 5, 3)
    for glu in ([False, True] if rows % 16 == 0 else [False]):
        for first in (0, 3):                      # rows at any byte
            want = ops.pack_int8(w[:, first:first + cols], scale, glu)
            got = ops.pack_int8(w.to(DEV)[:, first:first + cols], scale.to(DEV), glu)
            assert torch.equal(got.data.cpu(), want.data) and torch.equal(got.scales.cpu(), want.scales) and got.glu == glu
    apart = w[:, :cols].T.contiguous().to(DEV).T
    assert torch.equal(ops.pack_int8(apart, scale.to(DEV)).data.cpu(), ops.pack_int8(w[:, :cols], scale).data)


def test_weight_in_8_bits(ops):
    w = rnd(300, 500)
    packed = ops.quantize_weight_int8(w.to(torch.bfloat16).to(DEV))
    q, scale = plain_int8(w.to(torch.bfloat16).float())
    assert torch.equal(packed.unpack().cpu(), q) and torch.equal(packed.scale.cpu(), scale)


def test_refusals(ops):
    E = ops.KernelError
    a8 = ops.int8_rows(4, 64, DEV)
    (w, sw) = (t.to(DEV) for t in integers(32, 64, 1))
    packed, glu = ops.pack_int8(w, sw), ops.pack_int8(w, sw, glu=True)
    out, half = torch.empty(4, 32, device=DEV), torch.empty(4, 16, device=DEV)
    for call in (
            lambda: ops.quantize_int8(torch.zeros(4, 64, dtype=torch.float16, device=DEV), a8),
            lambda: ops.quantize_int8(torch.zeros(4, 63, device=DEV), a8),
            lambda: ops.quantize_int8(torch.zeros(4, 64), a8),
            lambda: ops.quantize_int8(torch.zeros(64, 4, device=DEV).T, a8),
            lambda: ops.add_rmsnorm_int8(torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV), torch.ones(64, device=DEV), 1e-6, a8),
            lambda: ops.add_rmsnorm_int8(torch.zeros(4, 64, device=DEV), torch.ones(32, device=DEV), 1e-6, a8),
            lambda: ops.add_rmsnorm_int8(torch.zeros(4, 64, device=DEV), torch.ones(64, device=DEV), 1e-6, a8, total=torch.zeros(4, 64, device=DEV)),
            lambda: ops.add_rmsnorm_int8(torch.zeros(4, 64, device=DEV), torch.ones(64, device=DEV), 1e-6, a8, y=torch.zeros(3, 64, device=DEV)),
            lambda: ops.int8_values(a8, torch.zeros(4, 64, dtype=torch.float64, device=DEV)),
            lambda: ops.gemm_int8(a8, packed, half),
            lambda: ops.gemm_int8(a8, packed, out.double()),
            lambda: ops.gemm_int8(a8, packed, half, swiglu="silu"),
            lambda: ops.gemm_int8(a8, glu, out),
            lambda: ops.gemm_int8(a8, glu, half, torch.zeros(32, device=DEV), swiglu="silu"),
            lambda: ops.gemm_int8(a8, glu, half, accumulate=True, swiglu="silu"),
            lambda: ops.gemm_int8(a8, packed, out, torch.zeros(31, device=DEV)),
            lambda: ops.gemm_int8(a8, packed, out, accumulate=7),
            lambda: ops.gemm_int8(a8, packed, out, cut=2),                # one k block
            lambda: ops.gemm_int8(a8, packed, out, cut=9),
            lambda: ops.gemm_int8(a8, packed, out, cut=10),
            lambda: ops.gemm_int8(a8, packed, out, cut=19),
            lambda: ops.gemm_int8(a8, packed, out, cut=21),
            lambda: ops.gemm_int8(a8, packed, out, cut=501),              # more groups than rows
            lambda: ops.gemm_int8(a8, packed, out, cut=-64),
            lambda: ops.gemm_int8(ops.int8_rows(4, 48, DEV), packed, out),
            lambda: ops.gemm_int8(ops.Int8Rows(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)), packed, out)):
        with pytest.raises(E):
            call()
