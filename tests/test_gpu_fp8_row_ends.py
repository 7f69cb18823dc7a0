"""Rows in 8-bit floating point whose memory ends with their last value (GPU): their values, whatever the width."""
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 2, 3, 5, 6, 7, 8, 9, 12, 15, 17, 127, 129, 1003, 4097])
def test_values_of_rows_that_end_their_memory(ops, cols, dtype):
    """Rows of 16-byte strides the last of which has no room behind it: data * scale, equal bits."""
    for rows in (1, 3):
        stride = -(-cols // 16) * 16
        room = torch.full(((rows - 1) * stride + cols,), 0x7f, dtype=torch.uint8, device=DEV)
        data = room.view(torch.float8_e4m3fn).as_strided((rows, cols), (stride, 1))
        g = torch.Generator().manual_seed(cols)
        values = (100 * torch.randn(rows, cols, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
        data.copy_(values.to(DEV))
        scales = torch.zeros(rows, -(-cols // 512) * 4)
        blocks = -(-cols // 128)
        scales[:, :blocks] = 0.5 + torch.rand(rows, blocks, generator=g)
        rows8 = ops.Fp8Rows(data, scales.to(DEV))
        out = torch.full((rows, cols + 3), 9.0, dtype=dtype, device=DEV)
        ops.fp8_values(rows8, out[:, :cols])
        want = (values.float() * scales[:, :blocks].repeat_interleave(128, dim=1)[:, :cols]).to(dtype)
        assert torch.equal(out[:, :cols].cpu(), want) and (out[:, cols:] == 9).all()
