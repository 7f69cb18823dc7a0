"""Rows at the edges of what 8 bits and float32 say (GPU)."""
import math

import pytest
import torch

from tests.test_gpu_int8 import check_norm, integers, on_gpu, plain_int8, rnd, same

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    return o


@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_not_a_number_stays_one_through_every_epilogue(ops, rows, dtype):
    """A token whose row held an infinity or a NaN (scale NaN) and a weight row that did: their results are NaN, all others numbers."""
    dim, width = 256, 144
    (a, sa), (w, sw) = integers(rows, dim, 7), integers(width, dim, 8)
    sa[5], sw[17] = math.nan, math.nan
    a[5], w[17] = 0, 0
    want = torch.zeros(rows, width, dtype=torch.bool)
    want[5], want[:, 17] = True, True
    a8 = on_gpu(ops, a, sa)
    packed = ops.pack_int8(w.to(DEV), sw.to(DEV))
    bias = rnd(width).to(DEV)
    for kw in (dict(), dict(bias=bias), dict(accumulate=True), dict(accumulate=ops.EPILOGUE_RELU2), dict(bias=bias, accumulate=ops.EPILOGUE_RELU2)):
        out = torch.ones(rows, width, dtype=dtype, device=DEV)
        ops.gemm_int8(a8, packed, out, **kw)
        assert torch.equal(torch.isnan(out.cpu()), want), kw
    glu = ops.pack_int8(w.to(DEV), sw.to(DEV) * 0.1, glu=True)
    want = want[:, :width // 2] | want[:, width // 2:]           # gate row 17 (its unit), and every unit of the token
    for kind in ("silu", "gelu_tanh", "swish_clamped"):
        units = torch.ones(rows, width // 2, dtype=dtype, device=DEV)
        ops.gemm_int8(a8, glu, units, swiglu=ops.glu_descriptor(kind, 3.0))
        assert torch.equal(torch.isnan(units.cpu()), want), kind
    sw[17], sw[17 + width // 2] = 0.01, math.nan                 # ... and an up row
    w[17 + width // 2] = 0
    up = ops.pack_int8(w.to(DEV), sw.to(DEV) * 0.1, glu=True)
    for kind in ("silu", "gelu_tanh", "swish_clamped"):
        units = torch.ones(rows, width // 2, dtype=dtype, device=DEV)
        ops.gemm_int8(a8, up, units, swiglu=ops.glu_descriptor(kind, 3.0))
        assert torch.equal(torch.isnan(units.cpu()), want), kind


@pytest.mark.parametrize("dim", [48, 500, 4100, 17000])
def test_norm_of_rows_whose_products_leave_float32(ops, dim):
    spread = torch.exp(rnd(5, dim, seed=4))
    def norm(x, gain, eps):                                      # noqa: E306
        out = ops.int8_rows(x.shape[0], dim, DEV)
        ops.add_rmsnorm_int8(x.to(DEV), gain.to(DEV), eps, out)
        return out
    # no gain against values of any size: rows of zeros; less of it than float32 says exactly: zeros too, or (what a row of results below
    # 2^-100 may keep) numbers, which are then no further off than the step of their 8 bits and the spacing of float32 down there
    x = rnd(5, dim) * torch.tensor([[1.0], [3e8], [1e20], [1e30], [5e37]])
    for gain in (torch.zeros(dim), torch.zeros(dim).bfloat16(), torch.full((dim,), 1e-42), rnd(dim, seed=9) * 1e-38):
        out = norm(x, gain, 1e-6)
        v = x.double() / torch.sqrt((x.double() ** 2).mean(dim=1, keepdim=True) + 1e-6) * gain.double()
        got, scale = out.data.cpu().double(), out.scale.cpu().double()
        kept = scale.gt(0)
        assert torch.isfinite(scale).all() and got[~kept & gain.eq(0).all()].eq(0).all() and float(v.abs().max()) < 2.0 ** -100
        off = (got * scale[:, None] - v).abs()
        assert (off <= torch.where(kept, 0.51 * v.abs().amax(dim=1) / 127 + 127 * 2.0 ** -149, v.abs().amax(dim=1))[:, None]).all()
    # large gains against small values that reach over many powers of two: each value keeps its bits
    x = rnd(5, dim) * spread ** 4 * torch.tensor([[1e-3], [1e-6], [1e-9], [1e-20], [1e-30]])
    gain = 1e37 * (1 + 0.3 * rnd(dim, seed=2).clamp(-2, 2))
    check_norm(norm(x, gain, 0.0), x, gain, 0.0, dim)
    # small gains, and values below what a square says in float32
    x = rnd(5, dim) * torch.tensor([[1.0], [1e-10], [1e-25], [1e-33], [1e-36]])
    gain = 1e-25 * (1 + 0.3 * rnd(dim, seed=2))
    check_norm(norm(x, gain, 0.0), x, gain, 0.0, dim)
    gain = 1 + 0.3 * rnd(dim, seed=2)
    check_norm(norm(x, gain, 0.0), x, gain, 0.0, dim)
    # what leaves float32 as a value is not a number in 8 bits
    gain = torch.ones(dim)
    gain[dim // 2] = math.inf
    out = norm(rnd(5, dim) + 3, gain, 1e-6)
    assert torch.isnan(out.scale).all() and out.data.eq(0).all()


@pytest.mark.parametrize("dim", [32768, 32769, 40003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first", [0, 1])
def test_quantize_rows_too_wide_to_be_held(ops, dim, dtype, first):
    wide = (rnd(4, dim + 8) * torch.exp(rnd(4, 1, seed=3))).to(dtype)
    wide[1, first + dim - 1], wide[2] = math.nan, 0.0
    x = wide[:, first:first + dim]                               # (rows that begin at any value)
    out = ops.int8_rows(4, dim, DEV)
    ops.quantize_int8(wide.to(DEV)[:, first:first + dim], out)
    want_q, want_scale = plain_int8(x.float())
    assert torch.isnan(want_scale[1]) and want_scale[2] == 0
    assert torch.equal(out.data.cpu(), want_q) and same(out.scale.cpu(), want_scale)


def test_a_layer_adds_its_mixers_result_unrounded(tmp_path):
    """The residual stream is float32 and so is what is added to it, as in a bfloat16 model."""
    from jllm_serve_b200.engine import Engine
    from tests.tiny import TINY_A, make_model_folder
    with Engine(make_model_folder(TINY_A, 3, tmp_path), weights="int8", page_size=8, max_tokens_cached=128, max_batch_tokens=64, max_running=2,
                ctx=64) as engine:
        block = engine.runner.model.blocks[0]
        x = rnd(10, block.dim).to(DEV)
        y = (1 + 2.0 ** -12 * rnd(10, block.dim, seed=1)).to(DEV)
        block.mixer.forward = lambda rows8, out, batch, cache: out.copy_(y)
        block.feed_forward.forward = lambda rows8, out, batch: None
        want = x + y
        block.forward(x, None, None)
        assert torch.equal(x, want)
