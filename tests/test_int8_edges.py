"""What the 8-bit operators refuse and how they hand their arguments on, at the edges (CPU)."""
import pytest
import torch

from jllm_serve_b200.csrc import ops


@pytest.mark.parametrize("rows,cols", [(1, 2 ** 31 - 16), (1, 2 ** 31 - 8176), (2 ** 31 - 1, 16), (2 ** 31 - 8191, 1)])
def test_rows_that_32_bits_do_not_count_are_refused(rows, cols):
    """A thread steps from its last value past the row's end by as much as the row's threads hold: that has to stay below 2^31."""
    data = torch.empty((rows, -(-cols // 16) * 16), dtype=torch.int8, device="meta")[:, :cols]
    with pytest.raises(ops.KernelError):
        ops.Int8Rows(data, torch.empty(rows, device="meta"))


@pytest.mark.parametrize("rows,cols", [(1, 2 ** 31 - 8192), (2 ** 31 - 8192, 16)])
def test_the_largest_rows(rows, cols):
    rows8 = ops.Int8Rows(torch.empty((rows, cols), dtype=torch.int8, device="meta"), torch.empty(rows, device="meta"))
    assert rows8.shape == (rows, cols)
    # the furthest that the kernels' 32-bit counters go: a row's step, four rows of one group, a group of tokens
    assert cols - 1 + 1024 * 8 <= 2 ** 31 - 1 and rows + 255 <= 2 ** 31 - 1


def test_a_norm_does_not_drop_what_it_cannot_do():
    from types import SimpleNamespace

    from jllm_serve_b200.parts.norm import RmsNorm
    norm = RmsNorm(SimpleNamespace(eps=1e-6), 16, {"n.weight": torch.ones(16)}, "n.", None)
    x, rows8 = torch.zeros(2, 16), ops.int8_rows(2, 16, "cpu")
    for call in (lambda: norm.forward(x, torch.empty(2, 16), add=x),                      # no sum in front of a bfloat16 result
                 lambda: norm.forward(x, rows8, row_index=torch.zeros(2, dtype=torch.int32)),
                 lambda: norm.forward(x, rows8, rows=1)):
        with pytest.raises(ops.KernelError, match="8 bits"):
            call()


def test_scales_of_any_stride_are_packed_by_a_copy():
    """What lies apart is brought together first, so that nothing but a copy writes the packed weight's scales."""
    w, scale = torch.ones(5, 8, dtype=torch.int8), torch.arange(10.0)[::2]
    seen = []

    class Watch(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if "copy_" in str(func):
                seen.append((args[0].shape, args[1].is_contiguous()))
            return func(*args, **(kwargs or {}))
    with Watch():
        packed = ops.pack_int8(w, scale)
    assert torch.equal(packed.scale, scale) and ((5,), True) in [(tuple(s), c) for s, c in seen]
