"""Waits end by the clock (GPU): the limit that every kernel's waits on barriers have, made to run out once."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_wait_gives_up_after_its_two_seconds():
    """A barrier that never completes, and nothing but the clock to end the waits for it."""
    from jllm_serve_b200.csrc import ops
    ops.require_device()
    ops.check_kernel_errors()
    g = torch.Generator().manual_seed(3)
    a, w = torch.randn(128, 64, generator=g).bfloat16().to(DEV), (torch.randn(128, 64, generator=g) * 0.05).bfloat16().to(DEV)
    out, again = torch.zeros(128, 128, device=DEV), torch.zeros(128, 128, device=DEV)
    ops.gemm_tcgen05(a, w, out, tile_width=128)
    torch.cuda.synchronize()
    ops.gemm_tcgen05_starve_next(by_clock=True)
    began = time.monotonic()
    ops.gemm_tcgen05(a, w, again, tile_width=128)
    torch.cuda.synchronize()
    assert 1.9 < time.monotonic() - began < 6.0
    with pytest.raises(ops.KernelError, match="bounded wait ran out inside gemm_tcgen05"):
        ops.check_kernel_errors()
    ops.gemm_tcgen05(a, w, again, tile_width=128)
    torch.cuda.synchronize()
    ops.check_kernel_errors()
    assert torch.equal(out, again)
