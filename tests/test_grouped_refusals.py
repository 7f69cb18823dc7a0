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
