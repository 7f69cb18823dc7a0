"""What the operators of ragged groups refuse in front of a launch (CPU)."""
import pytest
import torch

from jllm_serve_b200.csrc import ops


@pytest.mark.parametrize("dim", [2 ** 32 + 8, 2 ** 31, ops.BLOCK_MOST + 1])
def test_answers_of_more_columns_than_32_bits_count(dim):
    """A launcher's 32 bits would take 2^32 + 8 columns for eight, and the rest of the result would stay as it was."""
    groups = ops.row_groups(2, 1, 3, "cpu")
    before = ops.launch_count
    with pytest.raises(ops.KernelError, match="columns"):
        ops.combine_groups(torch.empty(2, dim, dtype=torch.bfloat16, device="meta"), groups, torch.zeros(2, 1), torch.empty(2, dim, device="meta"))
    assert ops.launch_count == before


def test_a_bfloat16_product_of_one_weight_is_refused_by_the_library():
    """Nothing offers it, no cut is fitted to it and the bfloat16 kernels have no bias and no sum to add: the launcher says so before it asks for a device."""
    import ctypes
    rows = ops._BlockRows(4096, 0, 128, 4, 64, 0)
    weight = ops._BlockWeight(8192, 0, 1, 128, 64, 1, 0, 0)
    lib = ops.library()
    assert lib.jllm_gemm_grouped(ctypes.addressof(rows), ctypes.addressof(weight), 0, 0, 0, ops.F32, 16384, ops.F32, 128, 0, 0, 0, 0) != 0
    assert b"one weight is built for e4m3" in lib.jllm_last_error()
