"""Weights rounded to 8-bit floating point on a GPU: the same scales and bytes as the exact definition gives, and as without a GPU."""
import pytest
import torch

from tests.fp8_weight_cases import LARGEST, expected, weight_at_ties

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    yield o
    o.check_kernel_errors()


@pytest.mark.parametrize("largest", LARGEST)
def test_a_weight_at_the_ties_is_rounded_once(ops, largest):
    w = weight_at_ties(largest)
    want, scale = expected(w)
    packed = ops.quantize_weight_fp8(w.to(DEV))
    assert packed.scales[0, 0, 0].item() == scale
    assert torch.equal(packed.unpack()[0].float().cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,glu", [((1, 1), False), ((300, 700), False), ((272, 5000), True), ((5, 144, 260), True), ((2, 130, 70000), False)])
def test_bytes_and_scales_with_and_without_a_gpu(ops, shape, glu, dtype):
    g = torch.Generator().manual_seed(len(shape) + shape[-1])
    w = (torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(shape[-1], generator=g))).to(dtype)
    here, there = ops.quantize_weight_fp8(w, glu), ops.quantize_weight_fp8(w.to(DEV), glu)
    assert torch.equal(there.scales.cpu(), here.scales) and torch.equal(there.data.cpu(), here.data)
    scale = (torch.nn.functional.pad(w.double(), (0, -shape[-1] % 128, 0, -shape[-2] % 128)).unflatten(-2, (-1, 128)).unflatten(-1, (-1, 128)).abs()
             .amax(dim=(-3, -1)) / 448).float()          # (nothing here is as small as 2^-100)
    assert here.scales[..., 0, :scale.shape[-1]].flatten().tolist() == scale.reshape(-1, *scale.shape[-2:])[:, 0].flatten().tolist()


def test_rows_of_a_block_and_its_weight_agree(ops):
    """128 equal magnitudes at most: a weight whose rows are all one row rounds as the row does (`quantize_fp8`)."""
    g = torch.Generator().manual_seed(8)
    row = torch.randn(1, 1280, generator=g)
    rows8 = ops.fp8_rows(1, 1280, DEV)
    ops.quantize_fp8(row.to(DEV), rows8)
    packed = ops.quantize_weight_fp8(row.expand(128, 1280).contiguous().to(DEV))
    assert torch.equal(packed.scales[0, 0, :10], rows8.scale[0])
    assert torch.equal(packed.unpack()[0].view(torch.uint8), rows8.data.view(torch.uint8).expand(128, 1280))
