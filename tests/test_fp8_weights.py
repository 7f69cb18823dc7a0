"""Weights rounded to 8-bit floating point: one rounding, from the exact quotient by the rounded scale (CPU; `test_gpu_fp8_weights.py` has the same on a GPU)."""
import pytest
import torch

from jllm_serve_b200.csrc import ops
from tests.fp8_weight_cases import LARGEST, expected, weight_at_ties


@pytest.mark.parametrize("largest", LARGEST)
def test_a_weight_at_the_ties_is_rounded_once(largest):
    w = weight_at_ties(largest)
    want, scale = expected(w)
    packed = ops.quantize_weight_fp8(w)
    assert packed.scales[0, 0, 0].item() == scale
    assert torch.equal(packed.unpack()[0].float(), want)


def test_blocks_of_a_large_weight_are_the_blocks_alone():
    """Rows are taken some at a time: of 300 x 70,000 values 128 at a time."""
    w = torch.randn(300, 70000, generator=torch.Generator().manual_seed(1)) * torch.logspace(-3, 3, 300)[:, None]
    packed = ops.quantize_weight_fp8(w)
    values, scales = packed.unpack()[0].float(), packed.scales[0]
    for r, c in ((0, 0), (128, 69888), (256, 640)):
        part = w[r:r + 128, c:c + 128].contiguous()
        alone = ops.quantize_weight_fp8(part)
        assert torch.equal(alone.unpack()[0].float(), values[r:r + 128, c:c + 128]) and alone.scales[0, 0, 0] == scales[r // 8, c // 128]


def test_what_is_not_a_number_stays_so():
    w = torch.ones(130, 260)
    w[0, 0], w[129, 259], w[5, 200] = float("nan"), float("inf"), -0.0
    packed = ops.quantize_weight_fp8(torch.stack([w, torch.ones_like(w)]))
    values = packed.unpack().float() * packed.scales[:, [0, 16], :3].repeat_interleave(128, 1)[:, :130].repeat_interleave(128, 2)[:, :, :260]
    assert values[0, :128, :128].isnan().all() and values[0, 129, 256:].isnan().all() and values[0, :128, 128:256].isfinite().all() and (values[1] - 1).abs().max() < 1e-6
    assert torch.signbit(packed.unpack()[0, 5, 200].float())
