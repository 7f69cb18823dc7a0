"""Grouped products of offsets, orders and places that no grouping made (GPU): nothing behind the rows or outside the result is touched, and offsets that do not ascend
from 0 on are no pairs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MOST, LEAST = 2 ** 31 - 1, -2 ** 31


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    yield o
    o.check_kernel_errors()


OFFSETS = {"negative": [-1, 3, 5, 8, 9, 14], "least": [LEAST] * 6, "descending": [0, 9, 4, 4, 10, 12], "last below": [0, 2, 4, 6, 8, 7], "alternating": [MOST, LEAST, MOST, LEAST, 0, 3],
           "beyond": [0, 3, MOST, MOST, MOST, MOST], "later": [5, 6, 6, 7, 60, 61], "all one group's": [0, 0, 0, 0, 0, MOST], "none": [7] * 6}


def ascends(numbers):
    return numbers[0] >= 0 and all(a <= b for a, b in zip(numbers, numbers[1:]))


@pytest.mark.parametrize("what", list(OFFSETS))
@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("by_pair", [False, True])
def test_offsets_that_no_grouping_made(ops, what, kind, by_pair):
    rows, top, groups, n, k = 30, 2, 5, 140, 200
    pairs, m = rows * top, rows * top if by_pair else rows
    g = torch.Generator().manual_seed(4)
    weight, x = torch.randn(groups, n, k, generator=g).to(DEV), torch.randn(m, k, generator=g).to(DEV)
    if kind == "fp8":
        w, a = ops.quantize_weight_fp8(weight), ops.fp8_rows(m, k, DEV)
        ops.quantize_fp8(x, a)
    else:
        w, a = ops.pack_grouped(weight.to(torch.bfloat16)), x.to(torch.bfloat16)
    room = ops.row_groups(rows, top, groups, DEV)
    for order in (torch.full((pairs,), LEAST), torch.full((pairs,), MOST), torch.randint(LEAST, MOST, (pairs,), generator=g)):
        room.order.copy_(order.to(torch.int32))
        for cut in (0, 16111, 16121, 32121, 64121, 128211):
            room.offsets.copy_(torch.tensor(OFFSETS[what], dtype=torch.int64).to(torch.int32))
            held = torch.full((pairs + 300, n), 5.0, device=DEV)
            ops.gemm_grouped(a, w, room, held[100:100 + pairs], by_pair=by_pair, cut=cut)
            touched = (held != 5).any(dim=1)
            assert not touched[:100].any() and not touched[100 + pairs:].any()
            if ascends(OFFSETS[what]):
                first, last = (min(i, pairs) for i in (OFFSETS[what][0], OFFSETS[what][-1]))
                assert touched[100 + first:100 + last].all() and not touched[100:100 + first].any() and held.isfinite().all()
            else:
                assert not touched.any()
    ops.check_kernel_errors()


@pytest.mark.parametrize("groups", [1, 31, 33, 257, 1024])
def test_offsets_of_any_bits(ops, groups):
    rows, top, n, k = 40, 1, 16, 16
    g = torch.Generator().manual_seed(groups)
    w, a = ops.pack_grouped(torch.randn(groups, n, k, generator=g).to(torch.bfloat16).to(DEV)), torch.randn(rows, k, generator=g).to(torch.bfloat16).to(DEV)
    room = ops.row_groups(rows, top, groups, DEV)
    for turn in range(20):
        numbers = torch.randint(LEAST, MOST, (groups + 1,), generator=g) if turn % 2 else torch.randint(-3, rows + 3, (groups + 1,), generator=g)
        room.offsets.copy_(numbers.to(torch.int32))
        for cut in (0, 16121, 64121, 128211):
            held = torch.full((rows + 200, n), 5.0, device=DEV)
            ops.gemm_grouped(a, w, room, held[100:100 + rows], cut=cut)
            touched = (held != 5).any(dim=1)
            assert not touched[:100].any() and not touched[100 + rows:].any()
            assert ascends(numbers.tolist()) or not touched.any()
    ops.check_kernel_errors()


def test_places_of_any_bits(ops):
    """A place outside the answers is none."""
    rows, top, dim = 50, 3, 24
    g = torch.Generator().manual_seed(1)
    room = ops.row_groups(rows, top, 4, DEV)
    held = torch.full((rows * top + 200, dim), float("nan"), device=DEV)
    held[100:100 + rows * top] = 1
    for turn in range(6):
        place = torch.randint(LEAST, MOST, (rows, top), generator=g) if turn else torch.full((rows, top), rows * top)
        if turn > 3:
            place = torch.where(torch.rand(rows, top, generator=g) < 0.5, place, torch.randint(0, rows * top, (rows, top), generator=g))
        room.place.copy_(place.to(torch.int32))
        out = torch.full((rows, dim), 3.0, device=DEV)
        ops.combine_groups(held[100:100 + rows * top], room, torch.ones(rows, top, device=DEV), out)
        want = ((place >= 0) & (place < rows * top)).sum(dim=1, keepdim=True).float().expand(rows, dim)
        assert torch.equal(out.cpu(), want)
