"""Rows at the edges of what 8 bits and float32 say (GPU)."""
import math

import pytest
import torch

from tests.test_gpu_int8 import integers, on_gpu, rnd

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
