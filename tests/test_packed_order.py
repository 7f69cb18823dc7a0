"""What a product reads of its weight in front of its wait is written, or followed, by a copy when the weight is packed (CPU)."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from jllm_serve_b200.csrc import ops


class Watch(TorchDispatchMode):
    """The operators that ran and write, with what they were given."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if "copy_" in str(func) or not all(word not in str(func) for word in ("index", "gather", "fill", "zero", "clone", "mul", "div")):
            self.seen.append((str(func), args))
        return out


def ends_with_a_copy(seen):
    """A copy of neighbouring values of one type is no kernel."""
    name, args = seen[-1]
    return "copy_" in name and args[0].is_contiguous() and args[1].is_contiguous() and args[0].dtype == args[1].dtype and args[0].shape == args[1].shape


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("shape", [(32, 48), (400, 1000), (3, 160, 300)])
def test_an_8_bit_weight_ends_with_a_copy(shape, glu):
    data = torch.ones(shape).to(torch.float8_e4m3fn)
    scale = torch.rand(shape[:-2] + (-(-shape[-2] // 128), -(-shape[-1] // 128)))
    with Watch() as watch:
        packed = ops.pack_fp8(data, scale, glu)
    assert ends_with_a_copy(watch.seen)
    assert watch.seen[-1][1][0].data_ptr() == packed.scales.data_ptr() and torch.equal(packed.scales[..., :1, 0].flatten(), scale.reshape(-1, *scale.shape[-2:])[:, 0, 0])
    with Watch() as watch:
        ops.quantize_weight_fp8(torch.ones(shape), glu)
    assert ends_with_a_copy(watch.seen)


@pytest.mark.parametrize("shape", [(128, 64), (5, 8), (300, 200)])
def test_a_bfloat16_weight_ends_with_a_copy(shape):
    """(A plain matrix that a product is given is packed in front of it.)"""
    with Watch() as watch:
        ops.pack_weight(torch.ones(shape, dtype=torch.bfloat16))
    assert ends_with_a_copy(watch.seen)
