"""The scale of 128 values in 8-bit floating point for all 2^23 significands of float32 and for every power of two (GPU): the largest magnitude over 448, rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    yield o
    o.check_kernel_errors()


def scales_of(ops, largest):
    """The scales of blocks with these largest magnitudes [rows, blocks], which stand somewhere in their blocks, of either sign."""
    rows, blocks = largest.shape
    x = torch.zeros(rows, blocks, 128, device=DEV)
    at = (torch.arange(rows * blocks, device=DEV) * 37 % 128).view(rows, blocks, 1)
    x.scatter_(2, at, torch.where(at % 2 == 0, largest[..., None], -largest[..., None]))
    out = ops.fp8_rows(rows, blocks * 128, DEV)
    ops.quantize_fp8(x.view(rows, -1), out)
    values = out.data.float().view(rows, blocks, 128)
    assert values.gather(2, at).abs().eq(448).all() and values.count_nonzero() == rows * blocks
    return out.scale


def by_448(largest):
    return (largest.double() / torch.full((), 448, dtype=torch.float64, device=DEV)).float()


def test_every_significand(ops):
    """(m / 448 is 2^-28 of itself or further from a tie of float32's, so that float64's rounding in front decides nothing.)"""
    for part in range(8):
        bits = (127 << 23) + part * 2 ** 20 + torch.arange(2 ** 20, dtype=torch.int32, device=DEV)
        largest = bits.view(torch.float32).view(1024, 1024)
        assert torch.equal(scales_of(ops, largest), by_448(largest))


def test_every_power_of_two(ops):
    """From 2^-100, below which the scale stays, to the largest numbers."""
    g = torch.Generator(device=DEV).manual_seed(3)
    exponent = torch.arange(27, 255, dtype=torch.int32, device=DEV)[:, None]
    bits = (exponent << 23) | torch.randint(0, 2 ** 23, (228, 64), generator=g, device=DEV).to(torch.int32)
    largest = bits.view(torch.float32)
    assert torch.equal(scales_of(ops, largest), by_448(largest))
